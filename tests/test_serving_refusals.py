"""What the serving step's entry points refuse, before anything is launched (no GPU is touched)."""
import ctypes

import pytest

import parakeet_linear as pk

P = 1 << 20  # an aligned address that is never read: every call here is refused on the host


def status(name, *args):
    fn = getattr(pk.lib, name)
    got = fn(*args, None)
    assert got < 0 and pk.last_error(), name
    return got


SHAPE, ALIGN, ARG = -1, -2, -4


def norm(**kw):
    a = dict(kind=0, input=P, residual=P + (1 << 21), weight=P + (1 << 22), residual_out=P + (1 << 23), output=P + (1 << 24), scales=P + (1 << 25),
             rows=4, width=1024, epsilon=1e-5)
    a.update(kw)
    return status("pk_rms_norm_quantize", *a.values())


@pytest.mark.parametrize("want,kw", [
    (ARG, {"kind": 2}), (SHAPE, {"rows": -1}), (SHAPE, {"width": 0}), (SHAPE, {"width": 1020}), (SHAPE, {"width": 16392}),
    (ARG, {"epsilon": -1e-5}), (ARG, {"epsilon": float("nan")}), (ARG, {"epsilon": 2.0}), (ARG, {"input": None}), (ARG, {"weight": None}),
    (ARG, {"output": None}), (ARG, {"scales": None}), (ALIGN, {"input": P + 8}), (ALIGN, {"residual": P + (1 << 21) + 2}),
    (ALIGN, {"output": P + (1 << 24) + 4}), (ALIGN, {"scales": P + (1 << 25) + 2}), (ARG, {"residual_out": P + 2048}),
    (ARG, {"residual_out": P + (1 << 21) + 2048}), (ARG, {"output": P}), (ARG, {"output": P + (1 << 23)}),
    (ARG, {"residual_out": P + (1 << 22)}), (ARG, {"output": P + (1 << 22)}), (ARG, {"scales": P + (1 << 22) + 4}), (ARG, {"scales": P}),
    (ARG, {"scales": P + (1 << 21)}), (ARG, {"scales": P + (1 << 23)}), (ARG, {"scales": P + (1 << 24) + 4092}),
])
def test_norm(want, kw):
    assert norm(**kw) == want


@pytest.mark.parametrize("want,kw", [
    (SHAPE, {"m": 17}), (SHAPE, {"m": -1}), (SHAPE, {"n": -1}), (SHAPE, {"k": 0}), (SHAPE, {"k": 192}), (SHAPE, {"k": 65664}),
    (ARG, {"input": None}), (ARG, {"q": None}), (ARG, {"scales": None}), (ARG, {"zeros": None}), (ARG, {"output": None}),
    (ALIGN, {"input": P + 2}), (ALIGN, {"q": P + 4}), (ALIGN, {"scales": P + 1}), (ALIGN, {"output": P + 2}), (ALIGN, {"bias": P + 2}),
    (SHAPE, {"n": (1 << 30) + 1}), (ARG, {"output": P + (1 << 16)}), (ARG, {"output": P + (2 << 16) + 64 * 128 - 4}), (ARG, {"output": P + (3 << 16) + 252}),
    (ARG, {"output": P + (4 << 16)}), (ARG, {"output": P + (5 << 16) - 252}),
])
@pytest.mark.parametrize("int8", [False, True])
def test_gemv(want, kw, int8):
    a = dict(input=P + (1 << 16), q=P + (2 << 16), scales=P + (3 << 16), zeros=P + (4 << 16), bias=P + (5 << 16), output=P, fp32=1, m=1, n=64, k=256)
    a.update(kw)
    if int8:
        a = {"input": a.pop("input"), "input_scales": P, **a}
    assert status("pk_gemv_int4g128_a8" if int8 else "pk_gemv_int4g128", *a.values()) == want


def test_gemv_int8_needs_scales():
    assert status("pk_gemv_int4g128_a8", P, None, P, P, P, P, P, 0, 1, 64, 256) == ARG


def apart(*names):
    return {n: P + (i << 24) for i, n in enumerate(names)}


@pytest.mark.parametrize("want,kw", [
    (SHAPE, {"page_size": 24}), (SHAPE, {"page_size": 8}), (SHAPE, {"page_size": 512}), (SHAPE, {"requests": 0}), (SHAPE, {"requests": 4097}),
    (SHAPE, {"max_pages": 0}), (SHAPE, {"max_pages": 1 << 27}), (SHAPE, {"capacity": -1}), (SHAPE, {"free_capacity": -1}),
    (ARG, {"held": None}), (ARG, {"added": None}), (ARG, {"free": None}), (ARG, {"range": None}), (ARG, {"table": None}), (ARG, {"starts": None}),
    (ARG, {"lengths": None}), (ARG, {"slots": None}), (ARG, {"info": None}), (ALIGN, {"held": P + 2}), (ALIGN, {"positions": P + (8 << 24) + 1}),
    (ARG, {"lengths": P}), (ARG, {"starts": P + 16}), (ARG, {"slots": P + (2 << 24) + 4}), (ARG, {"info": P + (3 << 24)}),
])
def test_plan(want, kw):
    a = apart("held", "added", "free", "range")
    a["free_capacity"] = 64
    a.update({n: P + ((i + 4) << 24) for i, n in enumerate(("table", "starts", "lengths", "slots", "positions", "info"))})
    a.update(requests=8, max_pages=10, page_size=16, capacity=32)
    a.update(kw)
    assert status("pk_page_plan", *a.values()) == want


@pytest.mark.parametrize("want,kw", [
    (ARG, {"kind": 2}), (SHAPE, {"page_size": 48}), (SHAPE, {"kv_heads": 0}), (SHAPE, {"kv_heads": 257}), (SHAPE, {"head_dim": 96}),
    (SHAPE, {"pages": 0}), (SHAPE, {"pages": 1 << 27}), (SHAPE, {"tokens": -1}), (SHAPE, {"tokens": (1 << 21) + 1}), (SHAPE, {"key_stride": 1016}), (SHAPE, {"value_stride": 1 << 31}),
    (ARG, {"key": None}), (ARG, {"value": None}), (ARG, {"slots": None}), (ARG, {"key_cache": None}), (ARG, {"value_cache": None}),
    (ALIGN, {"key": P + 8}), (ALIGN, {"value_stride": 1028}), (ALIGN, {"value_cache": P + 8}), (ALIGN, {"slots": P + 2}),
])
def test_write(want, kw):
    a = dict(kind=0, key=P, key_stride=1024, value=P, value_stride=1024, slots=P, key_cache=P, value_cache=P, tokens=3, kv_heads=8, head_dim=128,
             page_size=16, pages=10, key_inverse_scale=1.0, value_inverse_scale=1.0)
    a.update(kw)
    assert status("pk_paged_cache_write", *a.values()) == want


@pytest.mark.parametrize("want,kw", [
    (ARG, {"kind": 3}), (SHAPE, {"page_size": 20}), (SHAPE, {"head_dim": 80}), (SHAPE, {"heads": 12}), (SHAPE, {"heads": 0}), (SHAPE, {"heads": 2048}),
    (SHAPE, {"kv_heads": 0}), (SHAPE, {"tokens": -1}), (SHAPE, {"tokens": (1 << 20) + 1}), (SHAPE, {"max_queries": 6}), (SHAPE, {"sequences": 4097}),
    (SHAPE, {"max_pages": 0}), (SHAPE, {"max_pages": (1 << 26) + 1}), (SHAPE, {"pages": 0}), (SHAPE, {"query_stride": 2040}),
    (SHAPE, {"output_stride": 0}), (ARG, {"query": None}), (ARG, {"key_cache": None}), (ARG, {"value_cache": None}), (ARG, {"block_table": None}),
    (ARG, {"query_starts": None}), (ARG, {"key_lengths": None}), (ARG, {"output": None}), (ALIGN, {"query": P + 8}), (ALIGN, {"query_stride": 2052}),
    (ALIGN, {"output": P + 4}), (ALIGN, {"key_cache": P + 8}), (ALIGN, {"block_table": P + 2}), (ALIGN, {"workspace": P + 8}),
    (ARG, {"workspace": None}), (ARG, {"workspace_bytes": 1000}), (ARG, {"max_queries": 1, "workspace": None}),
    (SHAPE, {"tokens": 1 << 20, "max_queries": 1 << 20, "heads": 128}),
])
def test_attention(want, kw):
    a = dict(kind=0, query=P, query_stride=2048, key_cache=P, value_cache=P, block_table=P, query_starts=P, key_lengths=P, output=P, output_stride=2048,
             tokens=5, max_queries=5, sequences=2, heads=16, kv_heads=8, head_dim=128, page_size=16, pages=10, max_pages=400, left=-1, right=0,
             scale=0.1, key_scale=1.0, value_scale=1.0, workspace=P, workspace_bytes=1 << 40)
    a.update(kw)
    assert status("pk_paged_attention", *a.values()) == want


def test_workspace_sizes_are_host_answers():
    assert pk.paged_attention_workspace_bytes(5, 5, 2, 16, 8, 128, 16, 400) >= 0
    assert pk.paged_attention_workspace_bytes(0, 0, 0, 16, 8, 128, 16, 400) >= 0
    for queries, kv, pages, none in ((5, 8, 48, True), (5, 8, 49, False), (5, 4, 48, True), (5, 2, 32, True), (5, 2, 33, False)):  # 10, 20, 40 rows
        assert (pk.paged_attention_workspace_bytes(5, queries, 2, 16, kv, 128, 16, pages) == 0) is none


@pytest.mark.parametrize("head_dim", [64, 128])
@pytest.mark.parametrize("page", [16, 256])
def test_workspace_sizes_hold_for_smaller_calls(head_dim, page):
    """A workspace for the largest step serves every step with fewer queries, sequences or pages."""
    queries, sequences, pages = (1, 2, 4, 8, 16, 40, 300), (1, 15, 16, 64, 4096), [n for n in (1, 2, 3, 4, 6, 20, 32, 33, 48, 49, 64, 96, 97, 200, 4000)]
    size = lambda q, s, p: pk.paged_attention_workspace_bytes(4096, q, s, 32, 8, head_dim, page, p)  # noqa: E731
    for axis, line in ((0, queries), (1, sequences), (2, pages)):
        for at in ((8, 16, 40), (40, 16, 33), (1, 1, 200), (300, 64, 4000), (4, 16, 3)):
            sizes = [size(*(at[:axis] + (x,) + at[axis + 1:])) for x in line]
            assert sizes == sorted(sizes), (axis, at)
    with pytest.raises(pk.PkError):
        pk.paged_attention_workspace_bytes(5, 5, 2, 16, 8, 100, 16, 400)


def test_empty_calls_return_before_a_launch():
    ok = lambda name, *args: getattr(pk.lib, name)(*args, None) == 0  # noqa: E731
    assert ok("pk_rms_norm_quantize", 0, None, None, None, None, None, None, 0, 1024, 1e-5)
    assert ok("pk_gemv_int4g128", None, None, None, None, None, None, 0, 0, 64, 128)
    assert ok("pk_paged_cache_write", 0, None, 1024, None, 1024, None, None, None, 0, 8, 128, 16, 4, 1.0, 1.0)
    assert ok("pk_paged_attention", 0, None, 1024, None, None, None, None, None, None, 1024, 0, 0, 0, 8, 8, 128, 16, 4, 4, -1, 0, 0.1, 1.0, 1.0, None,
              ctypes.c_uint64(0))
