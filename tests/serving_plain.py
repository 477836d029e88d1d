"""The serving step's operators from their definitions, in 64 bits, with bounds for what a kernel
that keeps sums in fp32 may be off.  Works on tensors of any device."""
import math

import torch

U16, U32 = 2.0**-11, 2.0**-24  # half a step of fp16 and fp32, relative
TINY16 = 2.0**-25              # half a step of fp16's smallest values


def e4m3_values(b):
    return b.view(torch.float8_e4m3fn).double()


def levels(q):
    """INT4-g128 words [n, k/8] -> levels [n, k]: byte b of word j holds k 8j + b (low nibble) and 8j + 4 + b (high)."""
    word = q.view(torch.int32).long() & 0xFFFFFFFF
    return torch.stack([(word >> (8 * (i % 4) + 4 * (i // 4))) & 15 for i in range(8)], -1).reshape(q.shape[0], -1)


def gemv(x, xs, q, scales, zeros, bias):
    """(y, bound of a fp32 kernel's error), both float64 [m, n]."""
    n, k = q.shape[0], q.shape[1] * 8
    w = (levels(q).double().view(n, -1, 128) - zeros.double()[..., None]) * scales.double()[..., None]
    w = w.view(n, k).t().contiguous()
    rows = x.double() if xs is None else x.double() * xs.double()[:, None]
    y, size = rows @ w, rows.abs() @ w.abs()
    if bias is not None:
        y, size = y + bias.double(), size + bias.double().abs()
    # fp16 rows: 128 products in a matrix sum (which may truncate: twice a rounding), a fused step per group, the waves'
    # parts (16 at most), row scale and bias; INT8 rows: the group sums are exact
    steps = k // 128 + 16 + 3
    return y, size * (steps * U32 + (0 if xs is not None else 2 * 128 * U32))


def rms_norm(x, r, w, eps):
    """(h, y) in float64."""
    h = x.double() + (0 if r is None else r.double())
    return h, h / (h.square().mean(1, keepdim=True) + eps).sqrt() * w.double()


def plan(held, added, free, begin, end, table, page, capacity):
    """Lists in, lists out: (table, starts, lengths, slots, positions, info)."""
    up = lambda t: -(-t // page)  # noqa: E731
    table = [list(row) for row in table]
    status = 0
    if any(h < 0 or a < 0 for h, a in zip(held, added)) or begin < 0:
        status |= 8
    if any(up(h + a) > len(table[0]) for h, a in zip(held, added)):
        status |= 2
    if sum(added) > capacity:
        status |= 4
    if sum(up(h + a) - up(h) for h, a in zip(held, added)) > min(end, len(free)) - begin:
        status |= 1
    if status:
        return table, [0] * (len(held) + 1), list(held), [-1] * capacity, [0] * capacity, [0, 0, status, 0]
    starts, slots, positions, at = [0], [], [], begin
    for r, (h, a) in enumerate(zip(held, added)):
        for c in range(up(h), up(h + a)):
            table[r][c] = free[at]
            at += 1
        for p in range(h, h + a):
            slots.append(table[r][p // page] * page + p % page if table[r][p // page] >= 0 else -1)
            positions.append(p)
        starts.append(starts[-1] + a)
    pad = capacity - len(slots)
    return (table, starts, [h + a for h, a in zip(held, added)], slots + [-1] * pad, positions + [0] * pad,
            [starts[-1], at - begin, 0, 0])


def attention(q, key, value, table, starts, lengths, left, right, scale, key_scale=1.0, value_scale=1.0):
    """(o, bound), float64, rows outside the sequences zero with bound 0.  Only the keys that a query sees are touched, so
    whatever the others hold cannot matter; keys of a page id outside the cache do not exist."""
    pages, kv, page, d = key.shape
    wide = lambda x: e4m3_values(x) if x.dtype == torch.uint8 else x.double()  # noqa: E731
    out, bound = torch.zeros(q.shape, dtype=torch.float64, device=q.device), torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    group = q.shape[1] // kv
    starts, lengths, table = starts.tolist(), lengths.tolist(), table.cpu()
    for r, length in enumerate(lengths):
        n = starts[r + 1] - starts[r]
        length = min(length, table.shape[1] * page)
        if n <= 0 or length <= 0:
            continue
        ids = table[r, : -(-length // page)]
        real = ((ids >= 0) & (ids < pages)).repeat_interleave(page)[:length].to(q.device)
        ids = ids.clamp(0, pages - 1).long().to(q.device)
        k = wide(key[ids]).transpose(1, 2).reshape(-1, kv, d)[:length] * key_scale
        v = wide(value[ids]).permute(0, 3, 1, 2).reshape(-1, kv, d)[:length] * value_scale
        j = torch.arange(length, device=q.device)
        at = length - n + torch.arange(n, device=q.device)[:, None]
        seen = real.expand(n, -1) & (j >= at - left if left >= 0 else j >= 0) & (j <= at + right if right >= 0 else j >= 0)
        hidden = ~seen.any(0)
        k, v = k.clone(), v.clone()
        k[hidden], v[hidden] = 0, 0  # seen by nobody
        for i in range(n):
            one = seen[i]
            if not one.any():
                continue
            ki, vi = k[one].permute(1, 0, 2), v[one].permute(1, 0, 2)  # [kv, keys, d]
            x = q[starts[r] + i].double().view(kv, group, d)
            p = torch.softmax(x @ ki.transpose(1, 2).contiguous() * scale, 2)
            o = p @ vi
            # scores: d products summed in fp32 (truncating at worst), three more roundings on |s|; exp2 and the sums; each
            # probability is rounded to fp16 (small ones by an absolute half step, next to a sum of 1 at least)
            size = (x.abs() @ ki.abs().transpose(1, 2).contiguous()).amax(2, keepdim=True)
            rel = U16 + 4 * (d + 3) * U32 * size * abs(scale) + (2 * ki.shape[1] + 64) * U32
            most = rel * (p @ vi.abs()) + rel * o.abs() + TINY16 * vi.abs().sum(1, keepdim=True) + U16 * o.abs() * (1 + rel) + TINY16
            out[starts[r] + i], bound[starts[r] + i] = o.view(-1, d), most.view(-1, d)
    return out, bound


def to_pages(k, v, page, table_row, key, value):
    """Writes float keys / values [length, kv, d] (already in the cache's type) into pages table_row of a cache."""
    for p in range(-(-k.shape[0] // page)):
        part_k, part_v = k[p * page:(p + 1) * page], v[p * page:(p + 1) * page]
        key[table_row[p], :, :part_k.shape[0]] = part_k.transpose(0, 1)
        value[table_row[p], :, :, :part_v.shape[0]] = part_v.permute(1, 2, 0)


def close(got, want, bound, what=""):
    """|got - want| <= bound everywhere (infinities and NaN in the same places)."""
    got, want = got.double(), want.double()
    odd = ~torch.isfinite(want)
    assert torch.equal(torch.isnan(got), torch.isnan(want)), f"{what}: NaN in other places"
    assert torch.equal(got[odd & ~torch.isnan(want)], want[odd & ~torch.isnan(want)]), f"{what}: other infinities"
    over = ((got - want).abs() - bound)[~odd]
    worst = float(over.max()) if over.numel() else 0.0
    assert worst <= 0 or math.isclose(worst, 0, abs_tol=0), f"{what}: {worst:.3g} beyond the bound"
