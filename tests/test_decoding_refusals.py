"""What the entry points between projection and cache, and behind the logits, refuse before anything is launched, and the
rotary frequencies (no GPU is touched)."""
import ctypes
import math

import pytest

import decoding_plain as plain
import parakeet_linear as pk
from test_serving_refusals import ALIGN, ARG, P, SHAPE, status

MB = 1 << 20


def at(i):
    return P + i * 64 * MB


def call(name, base, kw, want):
    a = dict(base)
    a.update(kw)
    assert status(name, *a.values()) == want


ROTATE = dict(query=at(0), query_stride=4096, key=at(1), key_stride=1024, query_weight=at(2), key_weight=at(3), positions=at(4), frequencies=at(5),
              query_out=at(6), query_out_stride=4096, key_out=at(7), key_out_stride=1024, tokens=33, heads=32, kv_heads=8, head_dim=128, rotary_dim=128,
              interleaved=0, amplitude=1.0, epsilon=1e-6)


@pytest.mark.parametrize("want,kw", [
    (SHAPE, {"tokens": -1}), (SHAPE, {"tokens": (1 << 21) + 1}), (SHAPE, {"heads": 0}), (SHAPE, {"heads": 1025}), (SHAPE, {"kv_heads": -1}),
    (SHAPE, {"kv_heads": 1025}), (SHAPE, {"head_dim": 16}), (SHAPE, {"head_dim": 120}), (SHAPE, {"head_dim": 272}), (SHAPE, {"rotary_dim": 8}),
    (SHAPE, {"rotary_dim": 144}), (SHAPE, {"rotary_dim": -16}), (SHAPE, {"query_stride": 4088}), (SHAPE, {"key_stride": 1016}),
    (SHAPE, {"query_out_stride": 1 << 31}), (SHAPE, {"key_out_stride": 0}), (ARG, {"epsilon": -1.0}), (ARG, {"epsilon": math.nan}),
    (ARG, {"epsilon": 1.5}), (ARG, {"amplitude": math.inf}), (ARG, {"amplitude": math.nan}), (ARG, {"query": None}), (ARG, {"key": None}),
    (ARG, {"query_out": None}), (ARG, {"key_out": None}), (ARG, {"positions": None}), (ARG, {"frequencies": None}), (ALIGN, {"query": at(0) + 8}),
    (ALIGN, {"key_out": at(7) + 2}), (ALIGN, {"query_weight": at(2) + 4}), (ALIGN, {"positions": at(4) + 2}), (ALIGN, {"frequencies": at(5) + 4}),
    (ALIGN, {"query_stride": 4100}), (ARG, {"query_out": at(0) + 16}), (ARG, {"query_out": at(0), "query_out_stride": 4104}),
    (ARG, {"query_out": at(1)}), (ARG, {"key_out": at(0) + 4096}), (ARG, {"key_out": at(6) + 32 * 8192}), (ARG, {"query_out": at(2) - 16}),
    (ARG, {"key_out": at(4)}), (ARG, {"key_out": at(5) + 496}), (ARG, {"key_out": at(3)}),
    # queries and keys of the same rows, one of them in place
    (ARG, {"key": at(0), "kv_heads": 32, "key_stride": 4096, "key_out_stride": 4096, "query_out": at(0)})])
def test_head_norm_rotary(want, kw):
    call("pk_head_norm_rotary", ROTATE, kw, want)


STORE = dict(kind=0, query=at(0), query_stride=6144, key=at(0) + 8192, key_stride=6144, value=at(0) + 10240, value_stride=6144, query_weight=at(2),
             key_weight=at(3), positions=at(4), slots=at(5), frequencies=at(6), query_out=at(7), query_out_stride=4096, key_cache=at(8), value_cache=at(9),
             tokens=33, heads=32, kv_heads=8, head_dim=128, rotary_dim=64, interleaved=1, amplitude=1.0, epsilon=1e-6, page_size=16, pages=4,
             key_inverse_scale=1.0, value_inverse_scale=1.0)
CACHE = 4 * 16 * 1024 * 2


@pytest.mark.parametrize("want,kw", [
    (ARG, {"kind": 2}), (SHAPE, {"page_size": 48}), (SHAPE, {"kv_heads": 0}), (SHAPE, {"kv_heads": 257}), (SHAPE, {"head_dim": 96}), (SHAPE, {"pages": 0}),
    (SHAPE, {"pages": 1 << 27}), (SHAPE, {"tokens": -1}), (SHAPE, {"value_stride": 1016}), (SHAPE, {"rotary_dim": 144}), (ARG, {"epsilon": 2.0}),
    (ARG, {"value": None}), (ARG, {"slots": None}), (ARG, {"key_cache": None}), (ARG, {"value_cache": None}), (ARG, {"positions": None}),
    (ALIGN, {"value": at(0) + 10248}), (ALIGN, {"slots": at(5) + 1}), (ALIGN, {"value_cache": at(9) + 8}), (ALIGN, {"value_stride": 6148}),
    (ARG, {"value_cache": at(8) + CACHE - 16}), (ARG, {"key_cache": at(7) - CACHE + 16}), (ARG, {"key_cache": at(0) + 32 * 12288 + 10240 + 16}),
    (ARG, {"key_cache": at(4)}), (ARG, {"key_cache": at(5)}), (ARG, {"value_cache": at(6)}), (ARG, {"value_cache": at(2)}), (ARG, {"key_cache": at(3)}),
    (ARG, {"query_out": at(0) + 8192, "query_out_stride": 6144}), (ARG, {"query_out": at(0) + 10240, "query_out_stride": 6144}),
    (ARG, {"query_out": at(5) - 16})])
def test_head_norm_rotary_write(want, kw):
    call("pk_head_norm_rotary_write", STORE, kw, want)


SELECT = dict(kind=0, logits=at(0), stride=1030, scores=at(1), ended=at(2), out_scores=at(3), out_tokens=at(4), out_parents=at(5), out_ended=at(6),
              sequences=8, beams=4, vocab=1025, choices=4, end_token=0, workspace=at(7), workspace_bytes=1 << 30)


@pytest.mark.parametrize("want,kw", [
    (ARG, {"kind": 2}), (SHAPE, {"sequences": -1}), (SHAPE, {"sequences": 4097}), (SHAPE, {"beams": 0}), (SHAPE, {"beams": 33}), (SHAPE, {"vocab": 0}),
    (SHAPE, {"vocab": (1 << 20) + 1}), (SHAPE, {"choices": 0}), (SHAPE, {"choices": 65}), (SHAPE, {"stride": 1024}), (SHAPE, {"stride": 1 << 31}),
    (ARG, {"end_token": -2}), (ARG, {"end_token": 1025}), (ARG, {"end_token": -1}), (ARG, {"logits": None}), (ARG, {"scores": None}),
    (ARG, {"out_scores": None}), (ARG, {"out_tokens": None}), (ARG, {"out_parents": None}), (ARG, {"workspace": None}), (ARG, {"workspace_bytes": 100}),
    (ALIGN, {"logits": at(0) + 1}), (ALIGN, {"kind": 1, "logits": at(0) + 2}), (ALIGN, {"scores": at(1) + 2}), (ALIGN, {"workspace": at(7) + 8}),
    (ARG, {"out_scores": at(0) + 2060 * 31}), (ARG, {"out_tokens": at(1)}), (ARG, {"out_parents": at(2)}), (ARG, {"out_ended": at(2) + 31}),
    (ARG, {"out_tokens": at(3) + 124}), (ARG, {"workspace": at(5)}), (ARG, {"workspace": at(0)})])
def test_beam_select(want, kw):
    call("pk_beam_select", SELECT, kw, want)


@pytest.mark.parametrize("sequences,want", [(4096, SHAPE), (2049, SHAPE), (2048, ARG)])  # the last: only its missing outputs
def test_beam_select_threads_of_one_launch(sequences, want):
    call("pk_beam_select", SELECT, dict(sequences=sequences, beams=32, vocab=1 << 20, stride=1 << 20, out_scores=None), want)


@pytest.mark.parametrize("want,kw", [
    (SHAPE, {"sequences": 4097}), (SHAPE, {"sequences": -1}), (SHAPE, {"beams": 0}), (SHAPE, {"beams": 33}), (SHAPE, {"row": -1}),
    (SHAPE, {"row": (1 << 32) + 1}), (ARG, {"state": None}), (ARG, {"parents": None}), (ARG, {"output": None}), (ALIGN, {"parents": at(1) + 1}),
    (ARG, {"output": at(0) + 16}), (ARG, {"output": at(1)}), (ARG, {"output": at(0) - 16})])
def test_beam_reorder(want, kw):
    call("pk_beam_reorder", dict(state=at(0), parents=at(1), output=at(2), sequences=8, beams=4, row=1024), kw, want)


FORK = dict(parents=at(0), table=at(1), lengths=at(2), free=at(3), range=at(4), free_capacity=100, held=at(5), new_table=at(6), new_lengths=at(7),
            copies=at(8), freed=at(9), info=at(10), rows=8, max_pages=10, page_size=16, pages=500, workspace=at(11), workspace_bytes=1 << 20)


@pytest.mark.parametrize("want,kw", [
    (SHAPE, {"page_size": 24}), (SHAPE, {"rows": 0}), (SHAPE, {"rows": 4097}), (SHAPE, {"max_pages": 0}), (SHAPE, {"max_pages": (1 << 26) + 1}),
    (SHAPE, {"max_pages": 1 << 26, "page_size": 32}), (SHAPE, {"pages": 0}), (SHAPE, {"pages": 1 << 27}), (SHAPE, {"pages": 1 << 26, "page_size": 32}),
    (SHAPE, {"free_capacity": -1}), *[(ARG, {n: None}) for n in ("parents", "table", "lengths", "free", "range", "new_table", "new_lengths", "copies",
                                                                "freed", "info", "workspace")],
    *[(ALIGN, {n: FORK[n] + 2}) for n in ("parents", "table", "free", "new_table", "copies", "info")], (ALIGN, {"workspace": at(11) + 8}),
    (ARG, {"workspace_bytes": 100}), (ARG, {"new_table": at(1)}), (ARG, {"new_lengths": at(2)}), (ARG, {"freed": at(3) + 396}), (ARG, {"copies": at(0)}),
    (ARG, {"info": at(4)}), (ARG, {"freed": at(5) + 496}), (ARG, {"copies": at(6) + 316}), (ARG, {"workspace": at(9) + 1984})])
def test_page_fork(want, kw):
    call("pk_page_fork", FORK, kw, want)


@pytest.mark.parametrize("want,kw", [
    (SHAPE, {"capacity": -1}), (SHAPE, {"pages": -1}), (ARG, {"info": None}), (ARG, {"free": None}), (ARG, {"range": None}), (ALIGN, {"freed": at(1) + 2}),
    (ARG, {"free": at(0) - 4}), (ARG, {"freed": at(2) + 396}), (ARG, {"range": at(0) + 12}), (ARG, {"range": at(2)})])
def test_page_keep(want, kw):
    call("pk_page_keep", dict(info=at(0), freed=at(1), free=at(2), range=at(3), capacity=100, pages=100), kw, want)


@pytest.mark.parametrize("want,kw", [
    (SHAPE, {"count": -1}), (SHAPE, {"count": 65536}), (SHAPE, {"layers": -1}), (SHAPE, {"layers": 4097}), (SHAPE, {"pages": 0}),
    (SHAPE, {"pages": 1 << 27}), (SHAPE, {"bytes": 0}), (SHAPE, {"bytes": 1000}), (SHAPE, {"bytes": (1 << 24) + 16}), (ARG, {"copies": None}),
    (ARG, {"key": None}), (ARG, {"value": None}), (ALIGN, {"copies": at(0) + 2}), (ALIGN, {"key": at(1) + 8}), (ARG, {"value": at(1) + 1024}),
    (ARG, {"copies": at(1) + 64})])
def test_paged_cache_copy(want, kw):
    call("pk_paged_cache_copy", dict(copies=at(0), count=8, key=at(1), value=at(2), bytes=1024, pages=100, layers=3), kw, want)


def test_empty_calls_return_before_a_launch():
    ok = lambda name, *args: getattr(pk.lib, name)(*args, None) == 0  # noqa: E731
    assert ok("pk_head_norm_rotary", None, 4096, None, 1024, None, None, None, None, None, 4096, None, 1024, 0, 32, 8, 128, 128, 0, 1.0, 0.0)
    assert ok("pk_head_norm_rotary_write", *{**STORE, "tokens": 0, "query": None, "key_cache": None}.values())
    assert ok("pk_beam_select", *{**SELECT, "sequences": 0, "logits": None, "workspace": None, "workspace_bytes": ctypes.c_uint64(0)}.values())
    assert ok("pk_beam_reorder", None, None, None, 0, 4, 16) and ok("pk_beam_reorder", None, None, None, 4, 4, 0)
    assert ok("pk_paged_cache_copy", None, 0, None, None, 16, 4, 4)


def test_workspaces_hold_for_smaller_calls():
    size = pk.beam_select_workspace_bytes
    lines = ((1, 7, 64, 4096), (1, 4, 32), (1, 100, 1025, 16384, 16385, 131071, 1 << 20), (1, 4, 63, 64))
    for axis in range(4):
        for base in ((64, 8, 50000, 8), (1, 1, 1, 1), (4096, 32, 16384, 64)):
            sizes = [size(*(base[:axis] + (x,) + base[axis + 1:])) for x in lines[axis]]
            assert sizes == sorted(sizes)
    size, lines = pk.page_fork_workspace_bytes, ((1, 8, 1000, 4096), (1, 30, 500, 1 << 20), (1, 4096, 65536, 65537, 1 << 20, (1 << 27) - 1))
    for axis in range(3):
        for base in ((1, 1, 1), (64, 100, 5000), (4096, 500, 1 << 20), (8, 4, 1 << 18)):
            sizes = [size(*(base[:axis] + (x,) + base[axis + 1:])) for x in lines[axis]]
            assert sizes == sorted(sizes)
    with pytest.raises(pk.PkError):
        pk.page_fork_workspace_bytes(5000, 4, 4)
    with pytest.raises(pk.PkError):
        pk.beam_select_workspace_bytes(1, 33, 4, 4)
    with pytest.raises(ValueError):
        pk.beam_select_workspace_bytes(-1, 3, 4, 4)


@pytest.mark.parametrize("dim", [16, 64, 80, 128, 256])
@pytest.mark.parametrize("base", [10000.0, 500000.0])
@pytest.mark.parametrize("scaling,rest", [("plain", ()), ("linear", (4.0,)), ("base", (8.0,)), ("bands", (32.0, 1.0, 4.0, 8192)), ("bands", (2.0, 0.5, 100.0, 333)),
                                          ("ramp", (32.0, 1.0, 32.0, 4096)), ("ramp", (4.0, 5.0, 5.5, 2048)), ("ramp", (4.0, 1e-6, 1e6, 2048))])
def test_frequencies(dim, base, scaling, rest):
    words = pk.rotary_frequencies(dim, base, getattr(pk, "ROTARY_" + scaling.upper()), *rest, device="cpu").tolist()
    want = plain.frequencies(dim, base, scaling, *rest)
    assert len(words) == dim // 2
    for w, f in zip(words, want):
        # a power and some products in doubles; and the word is a whole number of 2^-64 turns, off by half of one
        assert abs(w / 2**64 * 2 * math.pi - f) <= f * 2.0**-46 + math.pi * 2.0**-64


@pytest.mark.parametrize("kw", [
    {"scaling": 5}, {"dim": 24}, {"dim": 0}, {"dim": 272}, {"base": 1.0}, {"base": math.nan}, {"base": math.inf}, {"scaling": 1, "factor": 0.5},
    {"scaling": 2, "factor": math.nan}, {"scaling": 3, "low": 0.0, "high": 1.0, "original": 10}, {"scaling": 3, "low": 2.0, "high": 2.0, "original": 10},
    {"scaling": 4, "low": 1.0, "high": math.inf, "original": 10}, {"scaling": 4, "low": 1.0, "high": 2.0, "original": 0}])
def test_frequencies_refused(kw):
    a = dict(dim=64, base=1e4, scaling=0, factor=1.0, low=0.0, high=0.0, original=0)
    a.update(kw)
    with pytest.raises(pk.PkError):
        pk.rotary_frequencies(*a.values(), device="cpu")
