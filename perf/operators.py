"""The operators of a decoder layer's serving step, one pass each: planning the
pages of a paged cache, the residual RMS norm with 8-bit rows, matrix-vector
products with INT4-g128 weights, writing keys and values into the cache, and the
attention of new tokens over it.

Each operator in its plain form (elementary torch operations in 32 bits), as the
library's calls (`own`), and from its definition in 64 bits (`exact`).  The
model's own sizes are width 1024, 8 heads of 128, joint 640 -> 1025 tokens + 5
durations, up to 45000 frames; the others are generic serving sizes.
"""
import math
import os
import sys

import torch

own = False

EPS = 1e-5
PROMPT = 2048  # tokens that one request adds in a step at most
LEFT_FRAMES = 128  # the encoder's local attention sees this many frames back


def _lib():
    path = os.path.join(os.getcwd(), "l4-parakeet-rs_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    import parakeet_linear

    return parakeet_linear


def listed():
    return [
        # Norm in front of a quantized linear: one token of a step at the model's width (latency alone),
        # every frame of one hour of audio (bandwidth).
        {"name": "norm_token", "op": "norm", "rows": 1, "width": 1024, "int8": False},
        {"name": "norm_hour", "op": "norm", "rows": 45000, "width": 1024, "int8": False},
        # 4-bit products of a step: the joint's 1030 outputs with fp32 scores for one frame (odd n, short k),
        # a wide projection for five streams on the norm's INT8 rows (weights larger than one L2).
        {"name": "gemv_joint", "op": "gemv", "m": 1, "n": 1030, "k": 640, "int8": False, "fp32": True},
        {"name": "gemv_wide", "op": "gemv", "m": 5, "n": 16384, "k": 8192, "int8": True, "fp32": False},
        # Pages of one step: eight streams of one token, a large server's step that mixes
        # single tokens with prompts (65536 slots, the last of them padding).
        {"name": "plan_streams", "op": "plan", "requests": 8, "page_size": 16, "most": 1500, "chunks": False, "capacity": 8},
        {"name": "plan_server", "op": "plan", "requests": 2000, "page_size": 16, "most": 8000, "chunks": True, "capacity": 65536},
        # New keys and values into the cache: one token of 61 streams in fp16, the prompts of a
        # step (a ragged 16000 tokens) in 8 bits.
        {"name": "write_tokens", "op": "write", "tokens": 61, "padding": 3, "kv_heads": 8, "head_dim": 128, "page_size": 16, "fp8": False, "chunk": 1},
        {"name": "write_prompts", "op": "write", "tokens": 16000, "padding": 384, "kv_heads": 8, "head_dim": 128, "page_size": 64, "fp8": True, "chunk": 1999},
        # Attention: one token of a short utterance at the model's heads (latency alone).
        {"name": "attend_token", "op": "attend", "sequences": 1, "queries": 1, "keys": 93, "ragged": False, "heads": 8, "kv_heads": 8,
         "head_dim": 128, "page_size": 16, "fp8": False, "left": -1, "right": 0},
        # One token of 64 ragged streams over long contexts, shared heads, 8-bit cache (bandwidth).
        {"name": "attend_streams", "op": "attend", "sequences": 64, "queries": 1, "keys": 8111, "ragged": True, "heads": 32, "kv_heads": 8,
         "head_dim": 128, "page_size": 64, "fp8": True, "left": -1, "right": 0},
        # One token over a very long context: few heads, so the keys have to be split.
        {"name": "attend_long", "op": "attend", "sequences": 1, "queries": 1, "keys": 120011, "ragged": False, "heads": 16, "kv_heads": 2,
         "head_dim": 128, "page_size": 128, "fp8": False, "left": -1, "right": 0},
        # Prompts in chunks over what is cached already (matrix products).
        {"name": "attend_chunks", "op": "attend", "sequences": 4, "queries": 777, "keys": 12007, "ragged": True, "heads": 32, "kv_heads": 8,
         "head_dim": 128, "page_size": 32, "fp8": False, "left": -1, "right": 0},
    ]


def _log(rng, lo, hi):
    return min(hi, int(lo * ((hi + 1) / lo) ** rng.random()))


def draw(rng):
    op = rng.choice(["norm", "norm", "gemv", "gemv", "gemv", "plan", "write", "attend", "attend", "attend", "attend"])
    if op == "norm":
        width = rng.choice([640, 1000, 1024, 2048, 2600, 4096, 5120, 8192])
        return {"op": op, "rows": _log(rng, 1, 45000 * 1024 // width), "width": width, "int8": rng.random() < 0.4}
    if op == "gemv":
        k = 128 * _log(rng, 3, 64)
        return {"op": op, "m": rng.randint(1, 16), "n": _log(rng, 100, 16384), "k": k, "int8": rng.random() < 0.5, "fp32": rng.random() < 0.25}
    if op == "plan":
        requests, chunks = _log(rng, 1, 2000), rng.random() < 0.5
        return {"op": op, "requests": requests, "page_size": rng.choice([16, 32, 64, 128, 256]), "most": _log(rng, 50, 8000), "chunks": chunks,
                "capacity": min(65536, requests * 32) if chunks else requests + rng.randint(0, 9)}
    kv_heads, head_dim, page_size = rng.choice([1, 2, 4, 8]), rng.choice([64, 128]), rng.choice([16, 32, 64, 128, 256])
    fp8 = rng.random() < 0.5
    if op == "write":
        tokens = _log(rng, 1, 16000)
        return {"op": op, "tokens": tokens, "padding": rng.randint(0, 20), "kv_heads": kv_heads, "head_dim": head_dim, "page_size": page_size,
                "fp8": fp8, "chunk": _log(rng, 1, tokens)}
    heads = kv_heads * rng.choice([1, 2, 3, 4, 5, 8])
    sequences = _log(rng, 1, 64)
    single = rng.random() < 0.5
    queries = 1 if single else _log(rng, 2, max(2, 777 * 4 // sequences))
    keys = queries + _log(rng, 1, min(120000, 64 * 8000 // sequences) if single else 12000)
    while sequences * heads * queries * keys > 4 * 32 * 777 * 12000 or sequences * keys > 64 * 8000:
        keys = (queries + keys) // 2  # at most the largest listed case's scores and keys
    left, right = rng.choice([(-1, 0), (-1, 0), (-1, 0), (LEFT_FRAMES, 0), (LEFT_FRAMES, 16), (-1, -1)])
    return {"op": op, "sequences": sequences, "queries": queries, "keys": keys, "ragged": rng.random() < 0.7, "heads": heads, "kv_heads": kv_heads,
            "head_dim": head_dim, "page_size": page_size, "fp8": fp8, "left": left, "right": right}


# ---- inputs -----------------------------------------------------------------------

def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _randn(g, *shape, scale=1.0):
    return (torch.randn(shape, generator=g, device="cuda") * scale).half()


def _ints(g, lo, hi, *shape):
    return torch.randint(lo, hi + 1, shape, generator=g, device="cuda", dtype=torch.int32)


def _e4m3(x):
    return x.clamp(-448.0, 448.0).to(torch.float8_e4m3fn)


def _prepare_norm(case, g):
    rows, width = case["rows"], case["width"]
    x, r = _randn(g, rows, width), _randn(g, rows, width, scale=3.0)
    loud = _ints(g, 0, width - 1, max(1, width // 200)).long()  # a few channels carry most of the energy, as in trained models
    r[:, loud] *= 20
    w = (torch.rand(width, generator=g, device="cuda") + 0.5).half()
    return {"x": x, "r": r, "w": w, "r_out": torch.empty_like(x), "scales": torch.empty(rows, device="cuda"),
            "out": torch.empty((rows, width), dtype=torch.int8 if case["int8"] else torch.uint8, device="cuda")}


def _prepare_gemv(case, g):
    m, n, k = case["m"], case["n"], case["k"]
    w = torch.randn((n, k // 128, 128), generator=g, device="cuda") * 0.02
    lo, hi = w.amin(2).clamp(max=0), w.amax(2).clamp(min=0)
    scales = ((hi - lo) / 15).clamp(min=2.0**-14).half()
    zeros = (-lo / scales.float()).round().clamp(0, 15)
    q = ((w / scales.float()[..., None]).round() + zeros[..., None]).clamp(0, 15).to(torch.uint8).view(n, k // 8, 2, 4)
    packed = (q[:, :, 0] | (q[:, :, 1] << 4)).contiguous().view(torch.int32).view(n, k // 8)
    s = {"q": packed, "scales": scales, "zeros": zeros.half(), "bias": torch.randn(n, generator=g, device="cuda") * 0.1,
         "out": torch.empty((m, n), dtype=torch.float32 if case["fp32"] else torch.float16, device="cuda")}
    if case["int8"]:
        s["x"] = torch.randint(-127, 128, (m, k), generator=g, device="cuda", dtype=torch.int8)
        s["xs"] = torch.rand(m, generator=g, device="cuda") * 0.02 + 0.01
    else:
        s["x"] = _randn(g, m, k)
    return s


def _prepare_plan(case, g):
    requests, page, capacity = case["requests"], case["page_size"], case["capacity"]
    held = _ints(g, 0, case["most"], requests)
    if case["chunks"]:  # most requests add one token, some a prompt, a few nothing; together less than the capacity
        weight = torch.rand(requests, generator=g, device="cuda") ** 8
        added = (weight / weight.sum() * (capacity - 2 * requests)).clamp(min=0, max=PROMPT - 1).int() + _ints(g, 0, 1, requests)
    else:
        added = torch.ones(requests, dtype=torch.int32, device="cuda")
    have, want = (held + page - 1) // page, (held + added + page - 1) // page
    total, most = int(want.sum()), (case["most"] + PROMPT) // page + 2
    ids = torch.randperm(total + 7, generator=g, device="cuda").int()
    column = torch.arange(most, device="cuda")
    start = torch.cumsum(have, 0) - have
    table = torch.where(column < have[:, None], ids[(start[:, None] + column).clamp(max=total)], torch.zeros((), dtype=torch.int32, device="cuda"))
    free = ids[int(have.sum()):].contiguous()
    ints = lambda *shape: torch.zeros(shape, dtype=torch.int32, device="cuda")  # noqa: E731
    return {"held": held, "added": added, "free": free, "range": torch.tensor([3, free.numel()], dtype=torch.int32, device="cuda"),
            "table": table.contiguous(), "starts": ints(requests + 1), "lengths": ints(requests), "slots": ints(capacity),
            "positions": ints(capacity), "info": ints(4)}


def _cache(case, pages, g=None):
    """Key and value pages, as bytes where they hold e4m3; random where `g` is given."""
    kv, d, page = case["kv_heads"], case["head_dim"], case["page_size"]
    found = []
    for shape in ((pages, kv, page, d), (pages, kv, d, page)):
        if g is None:
            found.append(torch.zeros(shape, dtype=torch.uint8 if case["fp8"] else torch.float16, device="cuda"))
        else:
            x = torch.randn(shape, generator=g, device="cuda", dtype=torch.float16)
            found.append(_e4m3(x * 16).view(torch.uint8) if case["fp8"] else x)
    return found


def _prepare_write(case, g):
    tokens, kv, d, page, chunk = case["tokens"], case["kv_heads"], case["head_dim"], case["page_size"], case["chunk"]
    qkv = _randn(g, tokens + case["padding"], 2 * kv * d)  # key and value are slices of one projection's rows
    pages_each = (chunk + page - 1) // page + 1
    chunks = (tokens + chunk - 1) // chunk
    pages = chunks * pages_each + 3
    ids = torch.randperm(pages, generator=g, device="cuda")
    t = torch.arange(tokens, device="cuda")
    at = _ints(g, 0, page - 1, chunks).long()[t // chunk] + t % chunk
    slots = ids[t // chunk * pages_each + at // page] * page + at % page
    slots = torch.cat([slots, torch.full((case["padding"],), -1, device="cuda")]).int()
    key, value = _cache(case, pages)
    return {"k": qkv[:, : kv * d].unflatten(1, (kv, d)), "v": qkv[:, kv * d:].unflatten(1, (kv, d)), "slots": slots, "key": key, "value": value,
            "inverse": (16.0, 20.0)}


def _prepare_attend(case, g):
    sequences, most, page, d = case["sequences"], case["queries"], case["page_size"], case["head_dim"]
    if case["ragged"]:
        count = _ints(g, (most + 1) // 2, most, sequences)
        length = count + (torch.rand(sequences, generator=g, device="cuda") * (case["keys"] - most + 1)).int()
    else:
        count = torch.full((sequences,), most, dtype=torch.int32, device="cuda")
        length = torch.full((sequences,), case["keys"], dtype=torch.int32, device="cuda")
    each = (length + page - 1) // page
    pages, columns = int(each.sum()) + 5, (case["keys"] + page - 1) // page
    ids = torch.randperm(pages, generator=g, device="cuda").int()
    column = torch.arange(columns, device="cuda")
    start = torch.cumsum(each, 0) - each
    table = torch.where(column < each[:, None], ids[(start[:, None] + column).clamp(max=pages - 1)], torch.zeros((), dtype=torch.int32, device="cuda"))
    starts = torch.zeros(sequences + 1, dtype=torch.int32, device="cuda")
    starts[1:] = torch.cumsum(count, 0)
    key, value = _cache(case, pages, g)
    q = _randn(g, sequences * most, case["heads"], d, scale=2.0)  # rows behind the last sequence's are padding
    return {"q": q, "key": key, "value": value, "table": table.contiguous(), "starts": starts, "lengths": length, "out": torch.zeros_like(q),
            "scale": 1 / math.sqrt(d), "key_scale": 0.0625 if case["fp8"] else 1.0, "value_scale": 0.0625 if case["fp8"] else 1.0}


def prepare(case, seed):
    s = globals()["_prepare_" + case["op"]](case, _gen(seed))
    s["case"] = dict(case)
    return s


# ---- plain forms ------------------------------------------------------------------

def _plain_norm(s):
    h = s["x"].float() + s["r"].float()
    s["r_out"].copy_(h)
    y = h * torch.rsqrt(h.square().mean(1, keepdim=True) + EPS) * s["w"].float()
    most = 127.0 if s["case"]["int8"] else 448.0
    scale = y.abs().amax(1) / most
    scale = torch.where(scale > 0, scale, torch.ones_like(scale))
    s["scales"].copy_(scale)
    y = y / scale[:, None]
    s["out"].copy_(y.round().clamp(-127, 127) if s["case"]["int8"] else _e4m3(y).view(torch.uint8))


def _levels(q):
    """INT4-g128 words [n, k/8] -> levels 0..15 as fp32 [n, k]: byte b of word j holds k 8j + b (low) and 8j + 4 + b (high)."""
    b = q.view(torch.uint8).view(q.shape[0], -1, 4)
    return torch.stack([b & 15, b >> 4], 2).reshape(q.shape[0], -1).float()


def _plain_gemv(s):
    n, k = s["q"].shape[0], s["q"].shape[1] * 8
    w = (_levels(s["q"]).view(n, k // 128, 128) - s["zeros"].float()[..., None]) * s["scales"].float()[..., None]
    y = s["x"].float() @ w.view(n, k).t()
    if s["case"]["int8"]:
        y = y * s["xs"][:, None]
    s["out"].copy_(y + s["bias"])


def _plain_plan(s):
    page, held, added, table = s["case"]["page_size"], s["held"], s["added"], s["table"]
    requests, columns, capacity = held.numel(), table.shape[1], s["slots"].numel()
    length = held + added
    have, want = (held + page - 1) // page, (length + page - 1) // page
    new_end, token_end = torch.cumsum(want - have, 0), torch.cumsum(added, 0)
    first = s["range"][0] + new_end - (want - have) - have  # free page of column c: free[first + c]
    short = new_end[-1] > s["range"][1] - s["range"][0]
    status = short.int() + 2 * (want.max() > columns).int() + 4 * (token_end[-1] > capacity).int()
    fits = status == 0
    last = s["free"].numel() - 1
    column = torch.arange(columns, device="cuda")
    new = (column >= have[:, None]) & (column < want[:, None]) & fits
    table.copy_(torch.where(new, s["free"][(first[:, None] + column).clamp(0, last)], table))
    t = torch.arange(capacity, device="cuda")
    r = torch.searchsorted(token_end, t, right=True).clamp(max=requests - 1)
    inside = (t < token_end[-1]) & fits
    at = held[r] + t - (token_end - added)[r]
    p = at // page
    ids = torch.where(p < have[r], table[r, p.clamp(0, columns - 1)], s["free"][(first[r] + p).clamp(0, last)])
    s["slots"].copy_(torch.where(inside, ids * page + at % page, torch.full_like(t, -1)))
    s["positions"].copy_(torch.where(inside, at, torch.zeros_like(at)))
    s["starts"][1:].copy_(token_end * fits)
    s["lengths"].copy_(torch.where(fits, length, held))
    s["info"].copy_(torch.stack([token_end[-1] * fits, new_end[-1] * fits, status, torch.zeros_like(status)]))


def _plain_write(s):
    page, d, tokens = s["case"]["page_size"], s["case"]["head_dim"], s["case"]["tokens"]
    slots = s["slots"][:tokens].long()
    k, v = s["k"][:tokens], s["v"][:tokens]
    if s["case"]["fp8"]:
        k, v = (_e4m3(x.float() * inverse).view(torch.uint8) for x, inverse in zip((k, v), s["inverse"]))
    s["key"][slots // page, :, slots % page] = k
    s["value"].transpose(2, 3)[slots // page, :, slots % page] = v


def _held(s, name, transposed):
    """The cache of every sequence, gathered through the table: fp32 [sequences, kv heads, columns * page size, head dim]."""
    x = s[name][s["table"].long()]
    x = (x.view(torch.float8_e4m3fn) if s["case"]["fp8"] else x).float() * (s["value_scale"] if transposed else s["key_scale"])
    x = x.permute(0, 2, 1, 4, 3) if transposed else x.permute(0, 2, 1, 3, 4)
    return x.reshape(x.shape[0], x.shape[1], -1, s["case"]["head_dim"])


def _plain_attend(s):
    case = s["case"]
    most, heads, kv, d = case["queries"], case["heads"], case["kv_heads"], case["head_dim"]
    starts, length = s["starts"], s["lengths"]
    count = starts[1:] - starts[:-1]
    k, v = _held(s, "key", False), _held(s, "value", True)
    sequences, keys = k.shape[0], k.shape[2]
    i, j = torch.arange(most, device="cuda"), torch.arange(keys, device="cuda")
    row = (starts[:-1, None] + i).clamp(max=s["q"].shape[0] - 1).long()
    q = s["q"][row].float().view(sequences, most, kv, heads // kv, d).permute(0, 2, 3, 1, 4).reshape(sequences * kv, -1, d)
    score = torch.bmm(q, k.view(sequences * kv, keys, d).transpose(1, 2).contiguous()).view(sequences, heads, most, keys) * s["scale"]
    at = (length - count)[:, None] + i
    seen = (j < length[:, None]).unsqueeze(1).expand(-1, most, -1)
    if case["left"] >= 0:
        seen = seen & (j >= (at - case["left"])[..., None])
    if case["right"] >= 0:
        seen = seen & (j <= (at + case["right"])[..., None])
    score.masked_fill_(~seen[:, None], -math.inf)
    top = score.amax(3, keepdim=True)
    score.sub_(torch.where(top > -math.inf, top, torch.zeros_like(top))).exp_()
    total = score.sum(3)
    v = torch.where((j < length[:, None])[:, None, :, None], v, torch.zeros((), device="cuda"))
    o = torch.bmm(score.view(sequences * kv, -1, keys), v.view(sequences * kv, keys, d)).view(sequences, heads, most, d)
    o = (o / torch.where(total > 0, total, torch.ones_like(total))[..., None]).transpose(1, 2)
    t = torch.arange(s["q"].shape[0], device="cuda")
    r = torch.searchsorted(starts[1:].long(), t, right=True).clamp(max=sequences - 1)
    s["out"].copy_(torch.where((t < starts[-1])[:, None, None], o[r, (t - starts[r]).clamp(max=most - 1)], s["out"]))


# ---- the library's calls --------------------------------------------------------------

def _own_norm(s):
    pk = _lib()
    kind = pk.NORM_INT8 if s["case"]["int8"] else pk.NORM_FP8
    pk.rms_norm_quantize(kind, s["x"], s["r"], s["w"], s["r_out"], s["out"], s["scales"], EPS)


def _own_gemv(s):
    pk = _lib()
    if s["case"]["int8"]:
        pk.gemv_int4g128_a8(s["x"], s["xs"], s["q"], s["scales"], s["zeros"], s["bias"], s["out"])
    else:
        pk.gemv_int4g128(s["x"], s["q"], s["scales"], s["zeros"], s["bias"], s["out"])


def _own_plan(s):
    _lib().page_plan(s["held"], s["added"], s["free"], s["range"], s["table"], s["starts"], s["lengths"], s["slots"], s["positions"], s["info"],
                     s["case"]["page_size"])


def _own_write(s):
    _lib().paged_cache_write(s["k"], s["v"], s["slots"], s["key"], s["value"], *s["inverse"])


def _own_attend(s):
    pk, case = _lib(), s["case"]
    if "workspace" not in s:
        size = pk.paged_attention_workspace_bytes(s["q"].shape[0], case["queries"], case["sequences"], case["heads"], case["kv_heads"],
                                                  case["head_dim"], case["page_size"], s["table"].shape[1])
        s["workspace"] = torch.empty(size, dtype=torch.uint8, device="cuda")
    pk.paged_attention(s["q"], s["key"], s["value"], s["table"], s["starts"], s["lengths"], s["out"], s["workspace"], max_queries=case["queries"],
                       left=case["left"], right=case["right"], scale=s["scale"], key_scale=s["key_scale"], value_scale=s["value_scale"])


def _outputs(s):
    op, case = s["case"]["op"], s["case"]
    held = lambda x: x.view(torch.float8_e4m3fn) if x.dtype == torch.uint8 else x  # noqa: E731
    if op == "norm":
        values = (s["out"] * s["scales"][:, None]).half() if case["int8"] else held(s["out"])
        return {"residual": s["r_out"], "values": values, "scales": s["scales"]}
    if op == "plan":
        return {name: s[name] for name in ("table", "starts", "lengths", "slots", "positions", "info")}
    if op == "write":
        return {"key": held(s["key"]), "value": held(s["value"])}
    return s["out"]


def run(state):
    op = state["case"]["op"]
    if own:
        globals()["_own_" + op](state)
    else:
        globals()["_plain_" + op](state)
    return _outputs(state)


# ---- from the definitions, in 64 bits -----------------------------------------------------

def _exact_norm(s):
    h = s["x"].double() + s["r"].double()
    y = h / (h.pow(2).sum(1, keepdim=True) / h.shape[1] + EPS).sqrt() * s["w"].double()
    scale = y.abs().max(1).values / (127 if s["case"]["int8"] else 448)
    return {"residual": h, "values": (y / scale[:, None]).round() * scale[:, None] if s["case"]["int8"] else y / scale[:, None], "scales": scale}


def _exact_gemv(s):
    q, n = s["q"].long(), s["q"].shape[0]
    y = torch.zeros(s["out"].shape, dtype=torch.float64, device="cuda")
    x = s["x"].double().view(s["x"].shape[0], -1, 8)
    zero, scale = (s[name].double().repeat_interleave(16, 1) for name in ("zeros", "scales"))
    for i in range(8):  # element i of every word of eight
        level = ((q >> (8 * (i % 4) + 4 * (i // 4))) & 15).double()
        y += x[:, :, i].contiguous() @ ((level - zero) * scale).t().contiguous()
    if s["case"]["int8"]:
        y *= s["xs"].double()[:, None]
    return y + s["bias"].double()


def _exact_write(s):
    found = []
    for name, x, inverse in zip(("key", "value"), (s["k"], s["v"]), s["inverse"] if s["case"]["fp8"] else (1.0, 1.0)):
        cache = torch.zeros(s[name].shape, dtype=torch.float64, device="cuda")
        rows = cache if name == "key" else cache.transpose(2, 3)
        real = s["slots"] >= 0
        at = s["slots"][real].long()
        rows[at // rows.shape[2], :, at % rows.shape[2]] = (x[real].double() * inverse).clamp(-448, 448) if s["case"]["fp8"] else x[real].double()
        found.append(cache)
    return {"key": found[0], "value": found[1]}


def _exact_attend(s):
    case = s["case"]
    kv, d, page = case["kv_heads"], case["head_dim"], case["page_size"]
    group = case["heads"] // kv
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    wide = lambda x: x.view(torch.float8_e4m3fn).double() if case["fp8"] else x.double()  # noqa: E731
    starts, lengths = s["starts"].tolist(), s["lengths"].tolist()
    for r, length in enumerate(lengths):
        ids = s["table"][r, : (length + page - 1) // page].long()
        first = length - (starts[r + 1] - starts[r])
        at = torch.arange(first, length, device="cuda")[:, None]
        j = torch.arange(length, device="cuda")[None]
        hidden = torch.zeros((at.shape[0], length), dtype=torch.bool, device="cuda")
        if case["left"] >= 0:
            hidden |= j < at - case["left"]
        if case["right"] >= 0:
            hidden |= j > at + case["right"]
        for h in range(kv):
            k = wide(s["key"][ids, h]).reshape(-1, d)[:length] * s["key_scale"]
            v = wide(s["value"][ids, h]).transpose(1, 2).reshape(-1, d)[:length] * s["value_scale"]
            for i in range(h * group, (h + 1) * group):
                q = s["q"][starts[r]:starts[r + 1], i].double()
                p = torch.softmax((q @ k.t() * s["scale"]).masked_fill(hidden, -math.inf), 1)
                out[starts[r]:starts[r + 1], i] = p @ v
    return out


def exact(case, seed):
    if case["op"] == "plan":  # whole numbers
        return None
    return globals()["_exact_" + case["op"]](prepare(case, seed))


# ---- what a pass cannot do without ---------------------------------------------------------

def work(case):
    op = case["op"]
    if op == "norm":
        n = case["rows"] * case["width"]
        return {"bytes": 7 * n + 4 * case["rows"] + 2 * case["width"], "flops": 8 * n}
    if op == "gemv":
        m, n, k = case["m"], case["n"], case["k"]
        return {"bytes": n * k // 2 + n * k // 32 + 4 * n + m * k * (1 if case["int8"] else 2) + m * n * (4 if case["fp32"] else 2),
                "flops": 2 * m * n * k}
    if op == "plan":
        requests, capacity, page = case["requests"], case["capacity"], case["page_size"]
        return {"bytes": 20 * requests + 8 * capacity + 8 * (capacity // page), "flops": 4 * requests + 8 * capacity}
    if op == "write":
        n = 2 * case["tokens"] * case["kv_heads"] * case["head_dim"]
        return {"bytes": n * (2 + (1 if case["fp8"] else 2)) + 4 * case["tokens"], "flops": n}
    sequences, queries, keys, d = case["sequences"], case["queries"], case["keys"], case["head_dim"]
    if case["ragged"]:  # on average
        queries, keys = queries * 0.75, queries * 0.75 + (keys - queries) / 2
    ahead = keys if case["right"] < 0 else case["right"]
    back = keys if case["left"] < 0 else case["left"]
    pairs = queries * max(1.0, min(keys, back + 1 + ahead, keys - queries / 2 + ahead))
    read = min(keys, back + queries + ahead)
    return {"bytes": sequences * (2 * read * case["kv_heads"] * d * (1 if case["fp8"] else 2) + 4 * queries * case["heads"] * d),
            "flops": 4 * d * case["heads"] * sequences * pairs}
