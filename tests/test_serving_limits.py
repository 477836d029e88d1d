"""Sizes that the serving step's entry points refuse because a kernel could not answer them (no GPU is touched)."""
import ctypes
import os
import random
import subprocess

import pytest

import parakeet_linear as pk
from conftest import PKG
from test_serving_refusals import ALIGN, ARG, P, SHAPE, status  # noqa: F401


@pytest.mark.parametrize("n,want", [(1 << 29, SHAPE), (1 << 30, SHAPE), ((1 << 29) - 1, ARG)])  # the last: only its missing output
def test_product_rows_of_one_launch(n, want):
    assert status("pk_gemv_int4g128", P, P, P, P, None, None, 1, 1, n, 128) == want
    assert status("pk_gemv_int4g128_a8", P, P, P, P, P, None, None, 1, 1, n, 128) == want


MB = 1 << 20
FREE = 1 << 30  # arrays below lie from here on, this far apart at least


def write_call(**kw):
    """Keys and values as slices of rows of 3 * 1024 elements; caches of 4 pages of 16 tokens, 8 heads of 128 (128 KB)."""
    a = dict(kind=0, key=FREE, key_stride=3080, value=FREE + 2048, value_stride=3080, slots=FREE + 16 * MB, key_cache=FREE + 32 * MB,
             value_cache=FREE + 48 * MB, tokens=33, kv_heads=8, head_dim=128, page_size=16, pages=4, key_inverse_scale=1.0, value_inverse_scale=1.0)
    a.update(kw)
    got = status("pk_paged_cache_write", *a.values())
    return got == ARG and b"overlap" in pk.lib.pk_last_error()


def attention_call(**kw):
    """Queries as slices of rows of 3080 elements, 16 heads of 128; the same caches; tables of 100 pages, shares."""
    a = dict(kind=0, query=FREE, query_stride=3080, key_cache=FREE + 32 * MB, value_cache=FREE + 48 * MB, block_table=FREE + 64 * MB,
             query_starts=FREE + 65 * MB, key_lengths=FREE + 66 * MB, output=FREE + 80 * MB, output_stride=2048, tokens=33, max_queries=33, sequences=2,
             heads=16, kv_heads=8, head_dim=128, page_size=16, pages=4, max_pages=100, left=-1, right=0, scale=0.1, key_scale=1.0, value_scale=1.0,
             workspace=FREE + 256 * MB, workspace_bytes=1 << 30)
    a.update(kw)
    got = status("pk_paged_attention", *a.values())
    return got == ARG and b"overlap" in pk.lib.pk_last_error()


CACHE = 4 * 16 * 1024 * 2


@pytest.mark.parametrize("kw", [
    {"value_cache": FREE + 32 * MB}, {"value_cache": FREE + 32 * MB + CACHE - 16}, {"key_cache": FREE + 48 * MB + 16}, {"key_cache": FREE},
    {"key_cache": FREE + 32 * 6160 + 2032}, {"value_cache": FREE - CACHE + 16}, {"slots": FREE + 32 * MB + 64}, {"slots": FREE + 48 * MB + CACHE - 4},
    {"slots": FREE + 32 * MB - 128}, {"value_cache": FREE + 6160 + 4080}])
def test_write_refuses_overlaps(kw):
    assert write_call(**kw)


@pytest.mark.parametrize("kw", [
    {"output": FREE + 16}, {"output": FREE, "output_stride": 4096}, {"output": FREE + 2 * 2040, "output_stride": 3080},
    {"output": FREE + 6160 * 32, "output_stride": 3080}, {"output": FREE - 6160 * 32 - 16, "output_stride": 3080},
    {"output": FREE - 6160 * 32 + 4096 - 16, "output_stride": 3080}, {"output": FREE + 32 * MB - 4096}, {"output": FREE + 48 * MB + CACHE - 16},
    {"output": FREE + 64 * MB + 784}, {"output": FREE + 65 * MB}, {"output": FREE + 66 * MB - 16}, {"output": FREE + 256 * MB + 4096},
    {"workspace": FREE + 32 * MB + 1024}, {"workspace": FREE + 48 * MB}, {"workspace": FREE + 64 * MB}, {"workspace": FREE + 60 * MB},
    {"workspace": FREE + 6160 * 31 + 4080}, {"workspace": FREE - MB}, {"query": FREE + 80 * MB + 2048, "query_stride": 2048}])
def test_attention_refuses_overlaps(kw):
    assert attention_call(**kw)


def test_overlaps_by_rows(tmp_path):
    """The answer for two sets of rows (csrc/pk_overlap.hpp) against a look at every pair of them, strides alike and not."""
    src, lib = tmp_path / "overlap.cpp", tmp_path / "overlap.so"
    src.write_text('#include "pk_overlap.hpp"\n'
                   'extern "C" int meet(int64_t s, int64_t w, int64_t n, int64_t at, int64_t s2, int64_t w2, int64_t n2) {\n'
                   '    const char* base = (const char*)(1ll << 32);\n'
                   '    return pk::overlap(pk::RowSet{base, s, w, n}, pk::RowSet{base + at, s2, w2, n2}) +\n'
                   '           2 * pk::overlap(pk::RowSet{base, s, w, n}, base + at, w2);\n}\n')
    subprocess.run(["g++", "-std=c++17", "-shared", "-fPIC", "-I", os.path.join(PKG, "csrc"), str(src), "-o", str(lib)], check=True)
    fn = ctypes.CDLL(str(lib)).meet
    fn.argtypes = [ctypes.c_int64] * 7
    rng, seen = random.Random(4), [0, 0]
    for _ in range(20000):
        w, n, w2, n2, at = rng.randint(1, 30), rng.randint(1, 6), rng.randint(1, 30), rng.randint(1, 6), rng.randint(-200, 200)
        s, s2 = w + rng.randint(0, 40), w2 + rng.randint(0, 40)
        if rng.random() < 0.6:
            s = s2 = max(s, s2)
        rows = [(i * s, i * s + w) for i in range(n)]
        others = [(at + i * s2, at + i * s2 + w2) for i in range(n2)]
        meet = any(a < d and c < b for a, b in rows for c, d in others)
        one = any(a < others[0][1] and others[0][0] < b for a, b in rows)
        assert fn(s, w, n, at, s2, w2, n2) == meet + 2 * one, (s, w, n, at, s2, w2, n2)
        seen[meet] += 1
    assert min(seen) > 5000


@pytest.mark.parametrize("kind,kw", [(0, {"scale": float("nan")}), (1, {"scale": float("inf")}), (1, {"key_scale": float("nan")}),
                                     (1, {"scale": 1e30, "key_scale": -1e30})])
def test_attention_needs_a_finite_scale(kind, kw):
    """Chunks took a NaN for 0, so that all keys counted alike."""
    a = dict(kind=kind, query=P, query_stride=2048, key_cache=P, value_cache=P, block_table=P, query_starts=P, key_lengths=P, output=P, output_stride=2048,
             tokens=0, max_queries=0, sequences=2, heads=16, kv_heads=8, head_dim=128, page_size=16, pages=10, max_pages=400, left=-1, right=0, scale=0.1,
             key_scale=1.0, value_scale=1.0, workspace=P, workspace_bytes=1 << 40)
    a.update(kw)
    assert status("pk_paged_attention", *a.values()) == ARG and b"finite" in pk.lib.pk_last_error()
