"""Sizes at which the calls around a decoding step's cache go from one form of a kernel to another: both sides, against the
plain forms."""
import random

import pytest

torch = pytest.importorskip("torch")

import test_gpu_rotary as rotary  # noqa: E402
from test_gpu_pages import Pool  # noqa: E402
from test_gpu_parity import pk  # noqa: E402, F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows,columns,spare", [
    (127, 20, 40), (128, 20, 40), (129, 20, 40), (128, 128, 40), (128, 129, 40), (113, 145, 40), (8, 60, (1 << 17) - 480), (8, 60, (1 << 17) - 479),
    (1024, 16, 40)])
def test_fork_in_one_launch_and_in_several(pk, rows, columns, spare):  # noqa: F811
    rng = random.Random(rows + columns)
    pool = Pool(rng, rows, columns, 16, spare=spare)
    for chance in (0.0, 0.1, 0.6):
        parents = [-1 if rng.random() < chance else min(rows - 1, r // 4 * 4 + rng.randrange(4)) for r in range(rows)]
        pool.go(pk, parents)
        pool.go(pk, parents, [int(rng.random() < 0.3) for _ in range(pool.pages)])


@pytest.mark.parametrize("tokens,heads,kv,d,r,page,how", [
    (6143, 2, 1, 64, 64, 32, "runs"), (6144, 2, 1, 64, 64, 32, "runs"), (6200, 2, 1, 128, 32, 16, "scattered"), (1535, 4, 4, 128, 64, 64, "runs"),
    (1536, 4, 4, 128, 64, 64, "runs"), (767, 9, 8, 128, 128, 64, "runs"), (768, 9, 8, 128, 128, 64, "runs"), (800, 8, 8, 64, 32, 16, "scattered"),
    (500, 16, 16, 64, 64, 32, "runs"), (30, 3, 256, 64, 64, 16, "runs")])
@pytest.mark.parametrize("fp8", [False, True])
def test_write_of_values_in_tiles_and_without(pk, tokens, heads, kv, d, r, page, how, fp8):  # noqa: F811
    rotary.test_write(pk, tokens, heads, kv, d, r, page, how, fp8, tokens % 2 == 0)
