"""What stands between projection and cache, and behind the logits, of a decoding step: from the definitions, in 64 bits or
whole numbers, with bounds for what a kernel that computes in fp32 may be off."""
import math

import torch

from serving_plain import TINY16, U16, U32

U8, TINY8 = 2.0**-4, 2.0**-10  # half a step of e4m3, relative and among its smallest values


def frequencies(dim, base, scaling="plain", factor=1.0, low=0.0, high=0.0, original=0):
    """Radians a position of each pair."""
    if scaling == "base":
        base = base * factor ** (dim / (dim - 2))
    f = [base ** (-2 * i / dim) for i in range(dim // 2)]
    if scaling == "linear":
        return [x / factor for x in f]
    if scaling == "bands":
        kept = [min(max((original * x / (2 * math.pi) - low) / (high - low), 0), 1) for x in f]
    elif scaling == "ramp":
        border = lambda turns: dim * math.log(original / (2 * math.pi * turns)) / (2 * math.log(base))  # noqa: E731
        first, last = max(math.floor(border(high)), 0), min(math.ceil(border(low)), dim - 1)
        kept = [1 - min(max((i - first) / max(last - first, 0.001), 0), 1) for i in range(dim // 2)]
    else:
        return f
    return [x * (k + (1 - k) / factor) for x, k in zip(f, kept)]


def phases(positions, words):
    """Radians of position * word, modulo a turn, exact until the last step: float64 [tokens x pairs]."""
    words = [w % 2**64 for w in words.tolist()]
    return torch.tensor([[(p * w % 2**64) / 2**64 * 2 * math.pi for w in words] for p in positions.tolist()], dtype=torch.float64).view(len(positions), -1)


def head_norm_rotary(x, weight, positions, words, interleaved, amplitude, eps):
    """(y, bound of what fp32 arithmetic may be off before the last rounding), both float64 [tokens, heads, head_dim]."""
    d = x.shape[2]
    y = x.double()
    rel = 0.0
    if weight is not None:
        mean = y.square().mean(2, keepdim=True) + eps
        y = torch.where(mean > 0, y / mean.sqrt(), torch.zeros_like(y)) * weight.double()
        # a sum of d squares over d, of which the root keeps half; reciprocal root within a step (2), two products; at most 6
        rel = ((d + 2) / 2 + 6) * U32
    bound = rel * y.abs()
    if words is None:
        return y, bound
    r = 2 * words.numel()
    angle = phases(positions, words).to(x.device)[:, None]
    c, s = amplitude * angle.cos(), amplitude * angle.sin()
    # sine and cosine: the argument (within pi / 4) is rounded three times, the series end within 2.6e-8, five fused steps
    # and the amplitude round, the phase loses its lower 32 bits
    off = abs(amplitude) * ((3 * 0.79 + 6) * U32 + 2.6e-8 + 2 * math.pi * 2.0**-32)
    out, most = y.clone(), bound.clone()
    a, b = (slice(0, r, 2), slice(1, r, 2)) if interleaved else (slice(0, r // 2), slice(r // 2, r))
    u, v = y[..., a], y[..., b]
    out[..., a], out[..., b] = u * c - v * s, v * c + u * s
    size = (u.abs() + v.abs()) * (off + abs(amplitude) * (rel + 3 * U32))
    most[..., a], most[..., b] = size, size
    return out, most


def in_half(y, bound):
    """Bound behind the rounding to fp16."""
    return bound + (y.abs() + bound) * U16 + TINY16


def in_e4m3(y, bound):
    return bound + (y.abs() + bound) * U8 + TINY8


def select(logits, scores, ended, end, choices):
    """Lists (scores in 64 bits, tokens, parents, ended) of the best candidates, and a bound for each score."""
    n, beams, vocab = logits.shape
    found = ([], [], [], [])
    for i in range(n):
        every = []
        for b in range(beams):
            have = float(scores[i, b])
            if not math.isfinite(have):
                continue
            if ended is not None and bool(ended[i, b]):
                every.append((-have, b * vocab + end, True))
                continue
            x = logits[i, b].double()
            top = x.max()
            if not torch.isfinite(top):  # NaN, infinity, or nothing that is allowed
                continue
            value = ((x - top) - (x - top).exp().sum().log()) + have  # (the logarithm beside a maximum of 2^53 and more would be lost)
            order = torch.argsort(x, descending=True, stable=True)[:choices]
            every += [(-float(value[t]), b * vocab + t, t == end) for t in order.tolist() if float(x[t]) > -math.inf]
        every.sort()
        every = every[:choices]
        left = choices - len(every)
        found[0].append([-e[0] for e in every] + [-math.inf] * left)
        found[1].append([e[1] % vocab for e in every] + [-1] * left)
        found[2].append([i * beams + e[1] // vocab for e in every] + [-1] * left)
        found[3].append([bool(e[2]) for e in every] + [False] * left)
    return found


# A term of a sum is exp2 of a difference that is rounded twice and scaled by a rounded constant: with d below the maximum its
# exponent is off by 3 d steps, and sum d exp(-d) / sum exp(-d) is at most ln(vocab) + 1 (20 for 2^24 tokens); the
# exponential itself two steps, a sum of eight terms seven.  The score's own rounding comes to it.
SCORE_STEPS = 3 * 20 + 2 + 7


def fork(parents, table, lengths, free, begin, end, page, pages, held=None):
    """Lists in, lists out: (table rows' entries, lengths, copies, freed, info)."""
    rows, columns = len(table), len(table[0])
    up = lambda n: -(-n // page)  # noqa: E731
    status = 0
    if begin < 0 or any(p < -1 or p >= rows for p in parents) or any(n < 0 or up(n) > columns for n in lengths):
        status = 8
    eldest, wanted = {}, []
    if not status:
        for r, p in enumerate(parents):
            if p >= 0:
                eldest.setdefault(p, r)
                if eldest[p] != r and lengths[p] % page and 0 <= table[p][lengths[p] // page] < pages:
                    wanted.append(r)
        if wanted and len(wanted) > min(end, len(free)) - begin:
            status = 1
    if status:
        return [list(t[:max(0, min(up(n), columns))]) for t, n in zip(table, lengths)], list(lengths), [[-1, -1]] * rows, [], [0, 0, status, 0]
    new, new_lengths, copies = [], [], []
    for r, p in enumerate(parents):
        n = lengths[p] if p >= 0 else 0
        row = list(table[p][:up(n)]) if p >= 0 else []
        pair = [-1, -1]
        if r in wanted:
            pair = [row[-1], free[begin + wanted.index(r)]]
            row[-1] = pair[1]
        new.append(row)
        new_lengths.append(n)
        copies.append(pair)
    listed = {p for t, n in zip(table, lengths) for p in t[:up(n)]}
    kept = {p for r in set(parents) - {-1} for p in table[r][:up(lengths[r])]}
    freed = sorted(p for p in listed - kept if 0 <= p < pages and not (held is not None and held[p]))
    return new, new_lengths, copies, freed, [sum(p >= 0 for p in parents), len(wanted), 0, len(freed)]
