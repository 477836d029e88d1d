"""Sizes at which the calls around a decoding step's cache go from one form of a kernel to another: both sides, against the
plain forms."""
import math
import random

import pytest

torch = pytest.importorskip("torch")

import test_gpu_rotary as rotary  # noqa: E402
from test_gpu_beams import Search, reordered  # noqa: E402
from test_gpu_pages import Pool  # noqa: E402
from test_gpu_parity import pk  # noqa: E402, F401
from test_gpu_serving import gen  # noqa: E402

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


@pytest.mark.parametrize("row", [1, 15, 16, 17, 31, 4095, 4096, 4097, 4111, 8207])
@pytest.mark.parametrize("beams", [1, 2, 8, 9, 32])
def test_reorder_in_place_of_units_and_single_bytes(pk, row, beams):  # noqa: F811
    """Rows of no unit, of units alone and with bytes behind them, in the first and last workgroup of a sequence; an unaligned
    state whose neighbours stay as they are."""
    n, g = 7, gen(row + beams)
    whole = torch.randint(0, 256, (n * beams * row + 32,), generator=g, device="cuda", dtype=torch.uint8)
    parents = torch.randint(0, beams, (n, beams), generator=g, device="cuda") + beams * torch.arange(n, device="cuda")[:, None]
    parents = torch.where(torch.rand((n, beams), generator=g, device="cuda") < 0.2, -1, parents).int()
    for shift in (0, 5):
        state = whole[16 + shift:16 + shift + n * beams * row].view(n, beams, row)
        before, want = whole.clone(), reordered(state, parents, state)
        pk.beam_reorder(state, parents, state)
        assert torch.equal(state, want)
        assert torch.equal(whole[:16 + shift], before[:16 + shift]) and torch.equal(whole[16 + shift + n * beams * row:], before[16 + shift + n * beams * row:])


@pytest.mark.parametrize("beams,vocab", [(17, 300), (20, 64), (32, 1024), (20, 1028)])
@pytest.mark.parametrize("choices", [16, 17, 32, 33])
@pytest.mark.parametrize("fp16", [False, True])
def test_select_of_short_rows_of_many_beams(pk, beams, vocab, choices, fp16):  # noqa: F811
    """More beams than the one launch takes, rows of up to a load a thread and of more: bounds of one wave and of all threads."""
    s = Search(pk, 3, beams, vocab, choices, fp16, seed=17)
    s.go()
    s.logits[0] = 0.25                      # equal logits, more than a list holds
    s.logits[1, :, choices // 2:] = -math.inf  # fewer candidates a row than choices
    s.logits[2] = s.logits[2].round()
    s.go()
