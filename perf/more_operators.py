"""The rest of a decoding step around the paged cache, one pass each: the norm of each query and key
head with the rotation by its position (with and without the write into the cache), the choice of the
next beams, states and pages that follow their beams, and copies of pages.

Each operator in its plain form (elementary torch operations in 32 bits, in 64 where angles of far
positions and candidates next to each other need them), as the library's calls (`own`), and from its
definition in 64 bits (`exact`).  The model's own sizes are 8 heads of 128, 1025 tokens, a prediction
network of two layers of 640; the others are generic serving sizes.
"""
import math
import os
import sys

import torch

own = False

EPS = 1e-6
FAR = 500000       # positions of long contexts
TRAINED = 8192     # positions before they were scaled
FACTOR = 32.0


def _lib():
    path = os.path.join(os.getcwd(), "l4-parakeet-rs_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    import parakeet_linear

    return parakeet_linear


def listed():
    return [
        # Queries and keys of one token at the model's heads (latency alone); the prompts of a step
        # (a ragged 16000 tokens) at far, scaled positions (bandwidth).
        {"name": "rotate_token", "op": "rotate", "tokens": 1, "heads": 8, "kv_heads": 8, "head_dim": 128, "rotary_dim": 128, "interleaved": False,
         "scaling": "plain", "norm": True, "chunk": 1},
        {"name": "rotate_prompts", "op": "rotate", "tokens": 16000, "heads": 32, "kv_heads": 8, "head_dim": 128, "rotary_dim": 128, "interleaved": False,
         "scaling": "ramp", "norm": True, "chunk": 1999},
        # The same with the write into the cache: one token of 61 streams into 8 bits, half of a head
        # rotated in neighbouring pairs; prompts into fp16.
        {"name": "store_tokens", "op": "store", "tokens": 61, "padding": 3, "heads": 32, "kv_heads": 8, "head_dim": 128, "rotary_dim": 64,
         "interleaved": True, "scaling": "bands", "norm": True, "chunk": 1, "page_size": 16, "fp8": True},
        {"name": "store_prompts", "op": "store", "tokens": 16000, "padding": 384, "heads": 32, "kv_heads": 8, "head_dim": 128, "rotary_dim": 128,
         "interleaved": False, "scaling": "plain", "norm": True, "chunk": 1999, "page_size": 64, "fp8": False},
        # Next beams: eight utterances of four beams over the model's tokens (fp32 scores of the joint),
        # 64 requests of eight beams over a wide vocabulary of odd size (bandwidth).
        {"name": "select_speech", "op": "select", "sequences": 8, "beams": 4, "vocab": 1025, "choices": 4, "fp16": False},
        {"name": "select_wide", "op": "select", "sequences": 64, "beams": 8, "vocab": 131071, "choices": 8, "fp16": True},
        # States behind their beams: two LSTM layers' hidden and cell rows of 640 (fp32) for 8 x 4 beams;
        # rows of a dense cache, 2 MB a beam.
        {"name": "reorder_lstm", "op": "reorder", "sequences": 8, "beams": 4, "row": 10240},
        {"name": "reorder_cache", "op": "reorder", "sequences": 16, "beams": 8, "row": 2097152},
        # Pages behind their beams: 8 x 4 beams of short utterances; 512 requests of eight beams over
        # long contexts (a table of 4096 rows).
        {"name": "fork_speech", "op": "fork", "sequences": 8, "beams": 4, "most": 450, "page_size": 16},
        {"name": "fork_server", "op": "fork", "sequences": 512, "beams": 8, "most": 8000, "page_size": 16},
        # The partly filled pages of a fork: 20 beams of one layer; 1500 beams through 12 layers of 8 heads.
        {"name": "copy_speech", "op": "copy", "copies": 32, "share": 0.6, "layers": 1, "kv_heads": 8, "head_dim": 128, "page_size": 16, "fp8": False},
        {"name": "copy_server", "op": "copy", "copies": 2048, "share": 0.7, "layers": 12, "kv_heads": 8, "head_dim": 128, "page_size": 16, "fp8": True},
    ]


def _log(rng, lo, hi):
    return min(hi, int(lo * ((hi + 1) / lo) ** rng.random()))


def draw(rng):
    op = rng.choice(["rotate", "store", "store", "select", "select", "reorder", "fork", "copy"])
    kv_heads, page_size, fp8 = rng.choice([1, 2, 3, 4, 8]), rng.choice([16, 32, 64, 128, 256]), rng.random() < 0.5
    if op in ("rotate", "store"):
        head_dim = rng.choice([64, 128]) if op == "store" else rng.choice([64, 80, 96, 128, 192, 256])
        heads = kv_heads * rng.choice([1, 2, 3, 4, 5])
        rotary_dim = rng.choice([head_dim, head_dim, 32, 48, 64])
        case = {"op": op, "tokens": _log(rng, 1, min(16000, 16000 * 40 * 128 // ((heads + kv_heads) * head_dim))), "heads": heads, "kv_heads": kv_heads,
                "head_dim": head_dim, "rotary_dim": rotary_dim, "interleaved": rng.random() < 0.4,
                "scaling": rng.choice(["plain", "linear", "base", "bands", "ramp"]), "norm": rng.random() < 0.75}
        case["chunk"] = _log(rng, 1, case["tokens"])
        if op == "store":
            case.update(padding=rng.randint(0, 20), page_size=page_size, fp8=fp8)
        return case
    if op == "select":
        beams, vocab, fp16 = rng.randint(1, 16), _log(rng, 100, 131072), rng.random() < 0.6
        choices = beams * rng.choice([1, 1, 2])
        most = 64 * 8 * 131071 // (beams * vocab * (1 if fp16 else 2)) * 8 // max(8, choices)
        return {"op": op, "sequences": _log(rng, 1, max(1, min(512, most))), "beams": beams, "vocab": vocab, "choices": choices, "fp16": fp16}
    if op == "reorder":
        beams, row = rng.randint(1, 16), rng.choice([1, 2, 4, 16, 16]) * _log(rng, 40, 131072)
        return {"op": op, "sequences": _log(rng, 1, max(1, min(512, 268000000 // (beams * row)))), "beams": beams, "row": row}
    if op == "fork":
        beams = rng.randint(1, 16)
        return {"op": op, "sequences": _log(rng, 1, 4096 // max(8, beams)), "beams": beams, "most": _log(rng, 50, 8000), "page_size": page_size}
    head_dim, layers = rng.choice([64, 128]), rng.randint(1, 12)
    page = page_size * kv_heads * head_dim * (1 if fp8 else 2)
    return {"op": op, "copies": _log(rng, 1, max(1, min(2048, 400000000 // (page * layers)))), "share": rng.choice([0.3, 0.7, 1.0]), "layers": layers,
            "kv_heads": kv_heads, "head_dim": head_dim, "page_size": page_size, "fp8": fp8}


# ---- inputs -----------------------------------------------------------------------

def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _ints(g, lo, hi, *shape):
    return torch.randint(lo, hi + 1, shape, generator=g, device="cuda", dtype=torch.int32)


def _e4m3(x):
    return x.clamp(-448.0, 448.0).to(torch.float8_e4m3fn)


def _scaling(case):
    """Arguments of the scaling beside (rotary_dim, base): (kind, factor, low, high, trained positions), and the amplitude."""
    kind = case["scaling"]
    low, high = {"bands": (1.0, 4.0), "ramp": (1.0, 32.0)}.get(kind, (0.0, 0.0))
    return (kind, 1.0 if kind == "plain" else FACTOR, low, high, TRAINED), 0.1 * math.log(FACTOR) + 1 if kind == "ramp" else 1.0


def _frequencies(case):
    """Radians a position of each pair, in 64 bits."""
    (kind, factor, low, high, trained), _ = _scaling(case)
    dim, base = case["rotary_dim"], 10000.0
    if kind == "base":  # a larger base that stretches the slowest pair by the factor
        base *= factor ** (dim / (dim - 2))
    i = torch.arange(dim // 2, dtype=torch.float64, device="cuda")
    f = base ** (-2 * i / dim)
    if kind == "linear":
        return f / factor
    if kind == "bands":  # by how often a pair turns over the trained positions
        kept = ((trained * f / (2 * math.pi) - low) / (high - low)).clamp(0, 1)
    elif kind == "ramp":  # the same borders, straight over the pairs' indices between them
        at = lambda turns: dim * math.log(trained / (2 * math.pi * turns)) / (2 * math.log(base))  # noqa: E731
        first, last = max(math.floor(at(high)), 0), min(math.ceil(at(low)), dim - 1)
        kept = 1 - ((i - first) / max(last - first, 0.001)).clamp(0, 1)
    else:
        return f
    return f * (kept + (1 - kept) / factor)


def _prepare_rotate(case, g):
    tokens, heads, kv, d = case["tokens"], case["heads"], case["kv_heads"], case["head_dim"]
    rows, chunk = tokens + case.get("padding", 0), case["chunk"]
    qkv = torch.randn((rows, heads + 2 * kv, d), generator=g, device="cuda")  # slices of one projection's rows
    qkv[:, :, _ints(g, 0, d - 1, 2).long()] *= 12  # a few loud channels, as in trained models
    qkv = (qkv * 0.7).half()
    chunks = (tokens + chunk - 1) // chunk
    t = torch.arange(tokens, device="cuda")
    most = FAR if case["scaling"] != "plain" else TRAINED
    positions = _ints(g, 0, most, chunks)[t // chunk] + t % chunk
    positions = torch.cat([positions, torch.zeros(rows - tokens, dtype=torch.int64, device="cuda")]).int()
    weight = lambda: (torch.rand(d, generator=g, device="cuda") * 1.5 + 0.25).half() if case["norm"] else None  # noqa: E731
    s = {"q": qkv[:, :heads], "k": qkv[:, heads:heads + kv], "v": qkv[:, heads + kv:], "qw": weight(), "kw": weight(), "positions": positions,
         "q_out": torch.zeros((rows, heads, d), dtype=torch.float16, device="cuda"), "f": _frequencies(case), "amplitude": _scaling(case)[1]}
    if case["op"] == "rotate":
        s["k_out"] = torch.zeros((rows, kv, d), dtype=torch.float16, device="cuda")
    if own:  # what a program keeps with its model
        (kind, *rest), _ = _scaling(case)
        pk = _lib()
        s["words"] = pk.rotary_frequencies(case["rotary_dim"], 10000.0, getattr(pk, "ROTARY_" + kind.upper()), *rest)
    return s


def _prepare_store(case, g):
    s = _prepare_rotate(case, g)
    tokens, kv, d, page, chunk = case["tokens"], case["kv_heads"], case["head_dim"], case["page_size"], case["chunk"]
    each, chunks = (chunk + page - 1) // page + 1, (tokens + chunk - 1) // chunk
    pages = chunks * each + 3
    ids = torch.randperm(pages, generator=g, device="cuda")
    t = torch.arange(tokens, device="cuda")
    at = _ints(g, 0, page - 1, chunks).long()[t // chunk] + t % chunk
    slots = ids[t // chunk * each + at // page] * page + at % page
    s["slots"] = torch.cat([slots, torch.full((case["padding"],), -1, device="cuda")]).int()
    kind = torch.uint8 if case["fp8"] else torch.float16
    s["key"] = torch.zeros((pages, kv, page, d), dtype=kind, device="cuda")
    s["value"] = torch.zeros((pages, kv, d, page), dtype=kind, device="cuda")
    s["inverse"] = (16.0, 20.0) if case["fp8"] else (1.0, 1.0)
    return s


def _prepare_select(case, g):
    n, beams, vocab, choices = case["sequences"], case["beams"], case["vocab"], case["choices"]
    logits = torch.randn((n, beams, vocab), generator=g, device="cuda") * 2
    likely = torch.randint(0, vocab, (n, beams, 6), generator=g, device="cuda")  # what the beam's next token may be
    logits.scatter_add_(2, likely, torch.rand((n, beams, 6), generator=g, device="cuda") * 12)
    logits.scatter_(2, torch.randint(1, vocab, (n, beams, 5), generator=g, device="cuda"), -math.inf)  # forbidden tokens
    scores = -torch.rand((n, beams), generator=g, device="cuda").cumsum(1) * 2 - 20 * torch.rand((n, 1), generator=g, device="cuda")
    ended = torch.rand((n, beams), generator=g, device="cuda") < 0.08
    make = lambda kind: torch.zeros((n, choices), dtype=kind, device="cuda")  # noqa: E731
    s = {"logits": logits.half() if case["fp16"] else logits, "scores": scores, "ended": ended, "end": 0, "out": make(torch.float32),
         "tokens": make(torch.int32), "parents": make(torch.int32), "out_ended": make(torch.bool)}
    if own:
        size = _lib().beam_select_workspace_bytes(n, beams, vocab, choices)
        s["workspace"] = torch.empty(size, dtype=torch.uint8, device="cuda")
    return s


def _parents(g, n, beams):
    """Parents as a search has them: the better beams have more children."""
    b = (torch.rand((n, beams), generator=g, device="cuda") ** 2 * beams).int().clamp(max=beams - 1)
    return (b.sort(1).values + beams * torch.arange(n, device="cuda")[:, None]).int()


def _prepare_reorder(case, g):
    shape = (case["sequences"], case["beams"], case["row"])
    kind = torch.float32 if case["row"] % 4 == 0 else torch.uint8  # bytes a row
    shape = shape[:2] + (case["row"] // (4 if kind is torch.float32 else 1),)
    state = torch.randn(shape, generator=g, device="cuda") if kind is torch.float32 else _ints(g, 0, 255, *shape).to(kind)
    return {"state": state, "parents": _parents(g, *shape[:2]), "out": torch.zeros_like(state)}


def _prepare_fork(case, g):
    n, beams, page, most = case["sequences"], case["beams"], case["page_size"], case["most"]
    rows, columns = n * beams, (most + page - 1) // page + 1
    length = _ints(g, 1, most, n)
    common = (length * (1 - 0.5 * torch.rand(n, generator=g, device="cuda"))).int() // page  # full pages of the prompt and what the beams agree on
    have = ((length + page - 1) // page).repeat_interleave(beams).long()
    common = torch.minimum(common, length // page).repeat_interleave(beams).long()
    first = torch.arange(rows, device="cuda") % beams == 0
    mine = torch.where(first, have, have - common)
    start = torch.cumsum(mine, 0) - mine
    total = int(mine.sum())
    lead = start.view(n, beams)[:, :1].expand(n, beams).reshape(rows)
    pages = rows * columns * (5 if beams >= 4 else 8) // 8 + 2 * rows + 9  # enough whatever the lengths
    ids = torch.randperm(pages, generator=g, device="cuda").int()
    c = torch.arange(columns, device="cuda")
    at = torch.where(first[:, None] | (c < common[:, None]), lead[:, None] + c, (start - common)[:, None] + c)
    table = torch.where(c < have[:, None], ids[at.clamp(max=pages - 1)], torch.zeros((), dtype=torch.int32, device="cuda")).int().contiguous()
    free = torch.cat([ids[:5], ids[total:]])  # the first five are taken
    parents = _parents(g, n, beams).view(rows)
    parents[torch.rand(rows, generator=g, device="cuda") < 0.02] = -1  # requests that are done
    ints = lambda *shape: torch.zeros(shape, dtype=torch.int32, device="cuda")  # noqa: E731
    s = {"parents": parents, "table": table, "lengths": length.repeat_interleave(beams).contiguous(), "free": free,
         "range": torch.tensor([5, free.numel()], dtype=torch.int32, device="cuda"), "pages": pages, "new_table": ints(rows, columns),
         "new_lengths": ints(rows), "copies": ints(rows, 2), "freed": ints(pages), "info": ints(4)}
    if own:
        s["workspace"] = torch.empty(_lib().page_fork_workspace_bytes(rows, columns, pages), dtype=torch.uint8, device="cuda")
    return s


def _prepare_copy(case, g):
    kv, d, page, count, layers = case["kv_heads"], case["head_dim"], case["page_size"], case["copies"], case["layers"]
    pages = 2 * count + 5
    ids = torch.randperm(pages, generator=g, device="cuda").int()
    real = torch.rand((count, 1), generator=g, device="cuda") < case["share"]
    copies = torch.where(real, torch.stack([ids[:count], ids[count:2 * count]], 1), torch.full((), -1, dtype=torch.int32, device="cuda"))
    shape = (layers, pages, kv * page * d)
    make = lambda: (torch.randint(0, 127, shape, generator=g, device="cuda", dtype=torch.uint8) if case["fp8"]  # noqa: E731
                    else torch.randn(shape, generator=g, device="cuda", dtype=torch.float16))
    return {"copies": copies.contiguous(), "key": make().view(layers, pages, kv, page, d), "value": make().view(layers, pages, kv, d, page)}


def prepare(case, seed):
    s = globals()["_prepare_" + case["op"]](case, _gen(seed))
    s["case"] = dict(case)
    return s


# ---- plain forms ------------------------------------------------------------------

def _rotated(s, x, weight):
    """Norm and rotation in fp32, from angles in 64 bits."""
    case = s["case"]
    x = x.float()
    if weight is not None:
        x = x * torch.rsqrt(x.square().mean(2, keepdim=True) + EPS) * weight.float()
    angle = s["positions"].double()[:, None] * s["f"]
    c, sn = (angle.cos() * s["amplitude"]).float()[:, None], (angle.sin() * s["amplitude"]).float()[:, None]
    r = case["rotary_dim"]
    if case["interleaved"]:
        u, v = x[..., 0:r:2], x[..., 1:r:2]
        turned = torch.stack([u * c - v * sn, v * c + u * sn], 3).flatten(2)
    else:
        u, v = x[..., :r // 2], x[..., r // 2:r]
        turned = torch.cat([u * c - v * sn, v * c + u * sn], 2)
    return torch.cat([turned, x[..., r:]], 2)


def _plain_rotate(s):
    s["q_out"].copy_(_rotated(s, s["q"], s["qw"]))
    s["k_out"].copy_(_rotated(s, s["k"], s["kw"]))


def _plain_store(s):
    page, tokens = s["case"]["page_size"], s["case"]["tokens"]
    s["q_out"][:tokens] = _rotated(s, s["q"], s["qw"])[:tokens].half()
    slots = s["slots"][:tokens].long()
    k, v = _rotated(s, s["k"], s["kw"])[:tokens], s["v"][:tokens].float()
    if s["case"]["fp8"]:
        k, v = (_e4m3(x * inverse).view(torch.uint8) for x, inverse in zip((k, v), s["inverse"]))
    else:
        k, v = k.half(), v.half()
    s["key"][slots // page, :, slots % page] = k
    s["value"].transpose(2, 3)[slots // page, :, slots % page] = v


def _plain_select(s):
    x, scores, end = s["logits"].double(), s["scores"].double(), s["end"]
    n, beams, vocab = x.shape
    top = x.amax(2, keepdim=True)
    total = (x - top).exp().sum(2, keepdim=True)
    x = (x - (top + total.log())) + scores[:, :, None]
    t = torch.arange(vocab, device="cuda")
    once = torch.where(t == end, scores[:, :, None], torch.full((), -math.inf, dtype=torch.float64, device="cuda"))
    x = torch.where(s["ended"][:, :, None], once, x).view(n, beams * vocab)
    index = torch.arange(beams * vocab, device="cuda")
    for j in range(s["case"]["choices"]):
        best = x.amax(1, keepdim=True)
        at = torch.where(x == best, index, beams * vocab).amin(1, keepdim=True)  # ties: the lowest
        found = best[:, 0] > -math.inf
        s["out"][:, j] = best[:, 0].float()
        s["tokens"][:, j] = torch.where(found, at[:, 0] % vocab, -1).int()
        row = torch.arange(n, device="cuda") * beams + at[:, 0] // vocab
        s["parents"][:, j] = torch.where(found, row, -1).int()
        s["out_ended"][:, j] = found & (s["ended"].view(-1)[row.clamp(max=n * beams - 1)] | (at[:, 0] % vocab == end))
        x.scatter_(1, at.clamp(max=beams * vocab - 1), -math.inf)


def _plain_reorder(s):
    state = s["state"]
    s["out"].view(-1, state.shape[2]).copy_(state.view(-1, state.shape[2])[s["parents"].view(-1).long()])


def _plain_fork(s):
    page, parents, table, length = s["case"]["page_size"], s["parents"].long(), s["table"], s["lengths"]
    rows, columns = table.shape
    r = torch.arange(rows, device="cuda")
    real = parents >= 0
    p = parents.clamp(min=0)
    child = torch.where(real, r, rows)
    eldest = torch.full((rows,), rows, dtype=torch.int64, device="cuda").scatter_reduce(0, p, child, "amin")
    new_length = torch.where(real, length[p], 0)
    last = new_length // page  # the partly filled page
    copied = real & (new_length % page > 0) & (eldest[p] != r)
    order = torch.cumsum(copied, 0)
    new = s["free"][(s["range"][0] + order - 1).clamp(0, s["free"].numel() - 1).long()]
    c = torch.arange(columns, device="cuda")
    inside = c < ((new_length + page - 1) // page)[:, None]
    to = torch.where((c == last[:, None]) & copied[:, None], new[:, None], table[p])
    s["new_table"].copy_(torch.where(inside, to, s["new_table"]))
    s["new_lengths"].copy_(new_length)
    none = p.clone().fill_(-1)
    source = torch.where(real, table[p, last.long().clamp(max=columns - 1)].long(), none)
    s["copies"].copy_(torch.where(copied[:, None], torch.stack([source, new.long()], 1), none[:, None]))
    # pages that a row listed and none does any more, lowest first
    listed = (c < ((length + page - 1) // page)[:, None])
    was = torch.zeros(s["pages"], dtype=torch.bool, device="cuda")
    was[table[listed].long()] = True
    kept = torch.zeros_like(was)
    kept[s["new_table"][inside].long()] = True
    back = was & ~kept
    place = torch.cumsum(back, 0)
    i = torch.arange(s["pages"], device="cuda")
    by_place = torch.zeros(s["pages"] + 1, dtype=torch.int32, device="cuda")
    by_place[torch.where(back, place - 1, s["pages"])] = i.int()
    s["freed"].copy_(torch.where(i < place[-1], by_place[:-1], s["freed"]))
    s["info"].copy_(torch.stack([real.sum(), order[-1], torch.zeros_like(order[-1]), place[-1]]))


def _plain_copy(s):
    real = s["copies"][:, 0] >= 0
    source, to = s["copies"][real].long().unbind(1)
    for x in (s["key"], s["value"]):
        x[:, to] = x[:, source]


# ---- the library's calls --------------------------------------------------------------

def _own_rotate(s):
    _lib().head_norm_rotary(s["q"], s["k"], s["qw"], s["kw"], s["positions"], s["words"], s["q_out"], s["k_out"],
                            interleaved=s["case"]["interleaved"], amplitude=s["amplitude"], epsilon=EPS)


def _own_store(s):
    _lib().head_norm_rotary_write(s["q"], s["k"], s["v"], s["qw"], s["kw"], s["positions"], s["slots"], s["words"], s["q_out"], s["key"], s["value"],
                                  *s["inverse"], interleaved=s["case"]["interleaved"], amplitude=s["amplitude"], epsilon=EPS)


def _own_select(s):
    _lib().beam_select(s["logits"], s["scores"], s["ended"], s["out"], s["tokens"], s["parents"], s["out_ended"], s["workspace"], end_token=s["end"])


def _own_reorder(s):
    _lib().beam_reorder(s["state"], s["parents"], s["out"])


def _own_fork(s):
    _lib().page_fork(s["parents"], s["table"], s["lengths"], s["free"], s["range"], s["new_table"], s["new_lengths"], s["copies"], s["freed"],
                     s["info"], s["workspace"], s["case"]["page_size"])


def _own_copy(s):
    _lib().paged_cache_copy(s["copies"], s["key"], s["value"])


def _outputs(s):
    op = s["case"]["op"]
    held = lambda x: x.view(torch.float8_e4m3fn) if x.dtype == torch.uint8 else x  # noqa: E731
    if op == "rotate":
        return {"query": s["q_out"], "key": s["k_out"]}
    if op == "store":
        return {"query": s["q_out"], "key": held(s["key"]), "value": held(s["value"])}
    if op == "select":
        return {"scores": s["out"], "tokens": s["tokens"], "parents": s["parents"], "ended": s["out_ended"]}
    if op == "reorder":
        return s["out"]
    if op == "fork":
        return {name: s[name] for name in ("new_table", "new_lengths", "copies", "freed", "info")}
    return {"key": held(s["key"]), "value": held(s["value"])}


def run(state):
    op = state["case"]["op"]
    if own:
        globals()["_own_" + op](state)
    else:
        globals()["_plain_" + op](state)
    return _outputs(state)


# ---- from the definitions, in 64 bits -----------------------------------------------------

def _exact_heads(s, x, weight):
    case, r = s["case"], s["case"]["rotary_dim"]
    y = x.double()
    if weight is not None:
        y = y / (y.pow(2).sum(2, keepdim=True) / y.shape[2] + EPS).sqrt() * weight.double()
    out = y.clone()
    phase = torch.polar(torch.full_like(s["f"], s["amplitude"])[None], s["positions"][:, None].double() * s["f"][None])
    for i in range(r // 2):
        a, b = (2 * i, 2 * i + 1) if case["interleaved"] else (i, i + r // 2)
        z = torch.complex(y[:, :, a].contiguous(), y[:, :, b].contiguous()) * phase[:, i, None]
        out[:, :, a], out[:, :, b] = z.real, z.imag
    return out


def _exact_rotate(s):
    return {"query": _exact_heads(s, s["q"], s["qw"]), "key": _exact_heads(s, s["k"], s["kw"])}


def _exact_store(s):
    real = s["slots"] >= 0
    q = _exact_heads(s, s["q"], s["qw"]) * real[:, None, None]
    found = {"query": q}
    for name, x, inverse in (("key", _exact_heads(s, s["k"], s["kw"]), s["inverse"][0]), ("value", s["v"].double(), s["inverse"][1])):
        cache = torch.zeros(s[name].shape, dtype=torch.float64, device="cuda")
        rows = cache if name == "key" else cache.transpose(2, 3)
        at = s["slots"][real].long()
        rows[at // rows.shape[2], :, at % rows.shape[2]] = (x[real] * inverse).clamp(-448, 448) if s["case"]["fp8"] else x[real]
        found[name] = cache
    return found


def _exact_select(s):
    n, beams, vocab = s["logits"].shape
    found = []
    for i in range(n):
        every = []
        for b in range(beams):
            if bool(s["ended"][i, b]):
                every.append(s["scores"][i, b:b + 1].double())
            else:
                p = torch.log_softmax(s["logits"][i, b].double(), 0) + s["scores"][i, b].double()
                every.append(p.topk(min(vocab, s["case"]["choices"])).values)
        every = torch.cat([torch.cat(every), torch.full((s["case"]["choices"],), -math.inf, dtype=torch.float64, device="cuda")])
        found.append(every.sort(descending=True).values[:s["case"]["choices"]])
    return {"scores": torch.stack(found), "tokens": None, "parents": None, "ended": None}


def exact(case, seed):
    if case["op"] in ("rotate", "store", "select"):
        return globals()["_exact_" + case["op"]](prepare(case, seed))
    return None  # whole numbers and copies


# ---- what a pass cannot do without ---------------------------------------------------------

def work(case):
    op = case["op"]
    if op in ("rotate", "store"):
        heads, kv, d, t = case["heads"], case["kv_heads"], case["head_dim"], case["tokens"]
        if op == "rotate":
            return {"bytes": t * (4 * (heads + kv) * d + 4), "flops": 10 * t * (heads + kv) * d}
        held = 1 if case["fp8"] else 2
        return {"bytes": t * (4 * heads * d + 2 * kv * d * (2 + held) + 8), "flops": 10 * t * (heads + kv) * d}
    if op == "select":
        rows = case["sequences"] * case["beams"]
        return {"bytes": rows * (case["vocab"] * (2 if case["fp16"] else 4) + 5) + case["sequences"] * case["choices"] * 13, "flops": 4 * rows * case["vocab"]}
    if op == "reorder":  # about 0.7 of the rows have children
        n = case["sequences"] * case["beams"] * case["row"]
        return {"bytes": int(1.7 * n), "flops": n // 4}
    if op == "fork":  # lengths are half the most on average
        rows = case["sequences"] * case["beams"]
        return {"bytes": 2 * 4 * rows * max(1, case["most"] // 2 // case["page_size"]) + 28 * rows, "flops": rows * (case["most"] // 2 // case["page_size"])}
    page = case["page_size"] * case["kv_heads"] * case["head_dim"] * (1 if case["fp8"] else 2)
    n = max(1, round(case["copies"] * case["share"])) * case["layers"] * page
    return {"bytes": 4 * n, "flops": n}
