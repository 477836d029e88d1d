"""Paged attention whose work is dealt in shares: several items a workgroup, one item over many of them."""
import pytest

torch = pytest.importorskip("torch")

from test_gpu_parity import pk  # noqa: E402, F401
from test_gpu_paged_attention import Case  # noqa: E402

pytestmark = pytest.mark.gpu

FEW_ROWS, CHUNKS = (512, 2), (256, 4)  # workgroups, and blocks that a share has at least


def blocks(case, left=-1, right=0):
    """Blocks that the batch is cut into, at least: keys of a (sequence, kv head, 16 rows) by 128 (e4m3: 256), or of a chunk's
    256 rows by 64."""
    group, total = case.heads // case.kv, 0
    for n, length in zip(case.counts, case.lengths_):
        for first in range(0, n * group, 16 if case.most * group <= 16 else 256):
            last = min(first + (16 if case.most * group <= 16 else 256), n * group) - 1
            lo = max(0, length - n + first // group - left) if left >= 0 else 0
            hi = min(length, length - n + last // group + right + 1) if right >= 0 else length
            keys = 64 if case.most * group > 32 else (256 if case.fp8 else 128)
            total += (-(-hi // keys) - lo // keys) * case.kv
    return total


@pytest.fixture(autouse=True)
def wide_tables():
    Case.wider = 6000
    yield
    Case.wider = 0


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("n", [1, 20])
def test_infinities_and_nan_stay_in_their_item(pk, fp8, n):  # noqa: F811
    """Infinities and NaN in one kv head's values of some sequences leave all other rows as they are, to the bit, whichever
    items stand before or behind them in a workgroup's share."""
    c = Case([(n, n + 3 + 89 * i % (600 if fp8 else 300)) for i in range(700)], heads=4, kv=2, fp8=fp8, seed=31)
    shares, least = FEW_ROWS if n == 1 else CHUNKS
    assert 2 * 700 > 2 * shares and blocks(c) > shares * least  # two items a share and more
    clean = c.run(pk).clone()
    for i in range(0, 700, 3):
        token = c.lengths_[i] - 1  # seen by the last row only
        p, off = int(c.table[i, token // c.page]), token % c.page
        c.value[p, i % 2, 5, off] = 0x7F if fp8 else (float("inf"), float("-inf"), float("nan"))[i // 3 % 3]
    for _ in range(3):
        got = c.run(pk).clone()
        for i in range(0, 700, 3):
            bad = got[int(c.starts[i + 1]) - 1, 2 * (i % 2):2 * (i % 2) + 2, 5]
            assert not torch.isfinite(bad).any() and (fp8 or i // 3 % 3 == 2 or (bad == (float("inf"), float("-inf"))[i // 3 % 3]).all())
            bad.copy_(clean[int(c.starts[i + 1]) - 1, 2 * (i % 2):2 * (i % 2) + 2, 5])
        assert torch.equal(got, clean)
