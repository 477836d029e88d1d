"""How the paged attention's work is cut and dealt (csrc/pk_paged_deal.hpp), compiled for the host: every row tile's
keys are in exactly one item, every block in exactly one share, also where a kv head has more than 2^31 blocks."""
import ctypes
import os
import random
import subprocess

import pytest

from conftest import PKG

SOURCE = r"""
#include "pk_paged_deal.hpp"
struct Args { int left, right, group, kv_heads; };
using namespace pk;
extern "C" long long per_head(int left, int right, int group, int rows, int length, int* tiles, int* pair) {
    const Args a{left, right, group, 1};
    const Pairs p = pairs_of(a, RowTile{0, rows, length, length - rows / group});
    *tiles = p.tiles;
    *pair = p.pair;
    return p.per_head;
}
extern "C" void span(int left, int right, int group, int rows, int length, long long offset, int* out) {
    const Args a{left, right, group, 1};
    const RowTile t{0, rows, length, length - rows / group};
    const Span s = span_at(a, t, pairs_of(a, t), offset);
    const int found[] = {s.kvh, s.tile, s.first, s.at, s.blocks};
    for (int i = 0; i < 5; ++i) out[i] = found[i];
}
// 0 where a walk over two kv heads meets each tile once, whole, with the blocks that its rows see; else a line number.
extern "C" int walk(int left, int right, int group, int rows, int length) {
    const Args a{left, right, group, 2};
    const RowTile t{0, rows, length, length - rows / group};
    const Pairs p = pairs_of(a, t);
    static int seen[2][4096];
    if (p.tiles > 4096) return __LINE__;
    for (int i = 0; i < p.tiles; ++i) seen[0][i] = seen[1][i] = 0;
    for (long long offset = 0; offset < 2 * p.per_head;) {
        const Span s = span_at(a, t, p, offset);
        if (s.kvh != offset / p.per_head || s.at != 0 || s.blocks <= 0 || s.tile >= p.tiles) return __LINE__;
        if (s.tile >= 0) {
            if (seen[s.kvh][s.tile]++) return __LINE__;
            int first = 0;
            if (chunk_blocks(a, t, s.tile, first) != s.blocks || first != s.first) return __LINE__;
            for (int r = s.tile * kChunkRows; r < (s.tile + 1) * kChunkRows && r < rows; ++r) {
                int lo = 0, hi = 0;
                window(a, t.first_pos + r / group, length, lo, hi);
                if (hi > lo && (lo < first * kTileKeys || hi > (first + s.blocks) * kTileKeys)) return __LINE__;
            }
        }
        for (int at = 1; at < s.blocks; at += 1 + s.blocks / 3) {  // from inside
            const Span in = span_at(a, t, p, offset + at);
            if (in.kvh != s.kvh || in.tile != s.tile || in.at != at || in.blocks != s.blocks) return __LINE__;
        }
        offset += s.blocks;
        if (offset > (s.kvh + 1) * p.per_head) return __LINE__;
    }
    for (int i = 0; i < p.tiles; ++i)
        if (!seen[0][i] || !seen[1][i]) return __LINE__;
    return 0;
}
template <int kShares, int kLeast> static int dealt(long long all) {
    if (share_begin<kShares, kLeast>(all, 0) != 0 || share_begin<kShares, kLeast>(all, kShares) != all) return __LINE__;
    for (int i = 0; i < kShares; ++i) {
        const long long from = share_begin<kShares, kLeast>(all, i), to = share_begin<kShares, kLeast>(all, i + 1);
        if (to < from || to - from > (all + kShares - 1) / kShares + kLeast) return __LINE__;
        for (const long long block : {from, from + (to - from) / 2, to - 1})
            if (from < to && share_of<kShares, kLeast>(all, block) != i) return __LINE__;
    }
    return 0;
}
extern "C" int deal(long long all) { return dealt<512, 2>(all) ? dealt<512, 2>(all) : dealt<256, 4>(all); }
"""


@pytest.fixture(scope="module")
def lib(tmp_path_factory):
    d = tmp_path_factory.mktemp("deal")
    (d / "deal.cpp").write_text("#include <initializer_list>\n" + SOURCE)
    subprocess.run(["g++", "-O2", "-std=c++17", "-shared", "-fPIC", "-I", os.path.join(PKG, "csrc"), str(d / "deal.cpp"), "-o", str(d / "deal.so")],
                   check=True)
    found = ctypes.CDLL(str(d / "deal.so"))
    found.per_head.restype = ctypes.c_longlong
    found.span.argtypes = [ctypes.c_int] * 5 + [ctypes.c_longlong, ctypes.c_void_p]
    found.deal.argtypes = [ctypes.c_longlong]
    return found


def window(pos, length, left, right):
    return (0 if left < 0 else max(0, pos - left)), max(0, length if right < 0 else min(length, pos + right + 1))


def tile_blocks(tile, rows, length, left, right, group):
    first = length - rows // group
    lo, _ = window(first + 256 * tile // group, length, left, right)
    _, hi = window(first + min(256 * tile + 255, rows - 1) // group, length, left, right)
    return lo // 64, max(1, -(-hi // 64) - lo // 64)


@pytest.mark.parametrize("left,right", [(-1, 0), (-1, -1), (128, 0), (128, 16), (60, -1), (0, 0), (777, 300)])
def test_each_tile_once(lib, left, right):
    rng = random.Random(left * 1000 + right)
    for _ in range(3000):
        group = rng.choice([1, 2, 3, 4, 5, 7, 8, 12, 16, 33, 66, 128, 257])
        n = max(1, rng.randint(1, 256 * rng.choice([1, 3, 9, 40])) // group)
        length = rng.choice([n, n + rng.randint(0, 3000), rng.randint(0, n)])
        assert lib.walk(left, right, group, n * group, length) == 0, (group, n, length)


@pytest.mark.parametrize("group,n,length", [(128, 65536, 5_000_000), (8, 1 << 20, 1 << 30), (1024, 8192, 1 << 30), (64, 131072, 300_000_001)])
@pytest.mark.parametrize("left,right", [(-1, 0), (-1, -1), (1 << 28, 0)])
def test_more_than_32_bits_of_blocks(lib, group, n, length, left, right):
    rows = group * n
    tiles, pair = ctypes.c_int(), ctypes.c_int()
    per_head = lib.per_head(left, right, group, rows, length, ctypes.byref(tiles), ctypes.byref(pair))
    assert tiles.value == rows // 256 and per_head == tiles.value // 2 * pair.value and per_head > 2**31
    out = (ctypes.c_int * 5)()
    for j in (0, 1, 2**31 // pair.value - 1, 2**31 // pair.value + 1, 2**32 // pair.value + 1, tiles.value // 2 - 1):
        if not 0 <= j < tiles.value // 2:
            continue
        at = j * pair.value
        first, blocks = tile_blocks(j, rows, length, left, right, group)
        for head in (0, 3):
            lib.span(left, right, group, rows, length, head * per_head + at + 1, out)
            assert list(out) == [head, j, first, 1, blocks]
            other, more = tile_blocks(tiles.value - 1 - j, rows, length, left, right, group)
            lib.span(left, right, group, rows, length, head * per_head + at + blocks, out)
            assert list(out) == [head, tiles.value - 1 - j, other, 0, more]


def test_shares(lib):
    rng = random.Random(3)
    for blocks in [*range(1, 40), *range(1000, 1100), *(rng.randint(1, 10 ** rng.randint(2, 12)) for _ in range(300))]:
        assert lib.deal(blocks) == 0, blocks
