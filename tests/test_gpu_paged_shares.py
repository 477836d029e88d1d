"""Paged attention whose work is dealt in shares: several items a workgroup, one item over many of them."""
import pytest

torch = pytest.importorskip("torch")

import serving_plain as plain  # noqa: E402
from test_gpu_parity import pk  # noqa: E402, F401
from test_gpu_paged_attention import Case  # noqa: E402

pytestmark = pytest.mark.gpu

FEW_ROWS, CHUNKS = (512, 2), (256, 4)  # workgroups, and blocks that a share has at least


def blocks(case, left=-1, right=0):
    """Blocks that the batch is cut into, at least: keys of a (sequence, kv head, 16 rows) by 128 (e4m3: 256), or of a chunk's
    256 rows by 64."""
    group, total = case.heads // case.kv, 0
    few = case.most * group <= 16  # (in a wide table)
    for n, length in zip(case.counts, case.lengths_):
        for first in range(0, n * group, 16 if few else 256):
            last = min(first + (16 if few else 256), n * group) - 1
            lo = max(0, length - n + first // group - left) if left >= 0 else 0
            hi = min(length, length - n + last // group + right + 1) if right >= 0 else length
            keys = (256 if case.fp8 else 128) if few else 64
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


# (new tokens, keys) whose blocks, more than the smallest shares hold, are dealt in proportion; windows for each
ONE = [(1, 120011)]
STREAMS = [(1, 1 + 1370 * i % 9001) for i in range(71)]
FEW = [(i % 3, 3 + 977 * i % 20011) for i in range(40)]
PROMPTS = [(300, 8111), (277, 6007), (5, 7000), (0, 900), (311, 9001)]
MANY = [(130 + i, 700 + 53 * i) for i in range(37)]
DEALT = [(ONE, 8, 4, (-1, 0)), (STREAMS, 8, 4, (-1, 0)), (FEW, 8, 4, (-1, 0)), (FEW, 8, 4, (5000, 0)), (PROMPTS, 32, 8, (-1, 0)), (PROMPTS, 24, 8, (-1, -1)),
         (PROMPTS, 32, 8, (2000, 0)), (PROMPTS, 20, 4, (3000, 16)), (MANY, 8, 4, (-1, 0))]


def dealt(shape, heads, kv, window, fp8):
    c = Case(shape, heads=heads, kv=kv, d=128, page=64, fp8=fp8, seed=7)
    shares, least = FEW_ROWS if c.most * heads // kv <= 16 else CHUNKS
    assert blocks(c, *window) > shares * least
    return c


def seen(c, r, window):
    """First and last key + 1 that each new token of sequence r sees."""
    n, length = c.counts[r], c.lengths_[r]
    at = torch.arange(length - n, length)
    lo = (at - window[0]).clamp(min=0) if window[0] >= 0 else torch.zeros_like(at)
    return lo, (at + window[1] + 1).clamp(max=length) if window[1] >= 0 else torch.full_like(at, length)


@pytest.mark.parametrize("shape,heads,kv,window", DEALT)
@pytest.mark.parametrize("fp8", [False, True])
def test_each_key_counts_once(pk, shape, heads, kv, window, fp8):  # noqa: F811
    """With equal scores an output is an average: feature f's values are 1 in the keys of every 128th block of 48 from f on,
    so that a block left out, or counted twice, shifts its feature by a twentieth at least."""
    c = dealt(shape, heads, kv, window, fp8)
    c.q.zero_()
    feature = torch.arange(128, device="cuda")
    for r, length in enumerate(c.lengths_):
        ids, j = c.table[r, :-(-length // c.page)].long(), torch.arange(-(-length // c.page) * c.page, device="cuda")
        one = ((j[:, None] // 48 % 128 == feature) & (j < length)[:, None]).half() / c.value_scale
        one = one.to(torch.float8_e4m3fn).view(torch.uint8) if fp8 else one
        c.value[ids] = one.view(-1, 1, c.page, 128).transpose(2, 3).expand(-1, kv, -1, -1)
    got = c.run(pk, *window).double().cpu()
    # p and 1 / sum are exact up to the rounding of sums of at most 2^11 terms in a row (a part's, then the parts')
    rel = plain.U16 + 2 * 2048 * plain.U32
    for r, (n, length) in enumerate(shape):
        lo, hi = (x[:, None] for x in seen(c, r, window))
        f = torch.arange(128)[None]
        upto = lambda x: x // (48 * 128) * 48 + (x % (48 * 128) - 48 * f).clamp(0, 48)  # noqa: E731 (keys below x of feature f)
        want = ((upto(hi) - upto(lo)).double() / (hi - lo))[:, None].expand(-1, heads, -1)
        off = (got[sum(c.counts[:r]):sum(c.counts[:r + 1])] - want).abs() - want * rel - plain.TINY16
        assert off.numel() == 0 or off.max() <= 0, (r, n, length, off.max(), off.argmax())


@pytest.mark.parametrize("shape,heads,kv,window", DEALT)
@pytest.mark.parametrize("fp8", [False, True])
def test_each_row_finds_its_key(pk, shape, heads, kv, window, fp8):  # noqa: F811
    """Keys of random signs, and each row's query that of a key it sees: its output is that key's value."""
    c = dealt(shape, heads, kv, window, fp8)
    if fp8:
        c.key[c.key != 0x7F] = (c.key[c.key != 0x7F] & 0x80) | 0x38  # +-1
    else:
        c.key[c.key == c.key] = torch.where(c.key[c.key == c.key] < 0, -1.0, 1.0).half()
    wide = lambda x: plain.e4m3_values(x) if fp8 else x.double()  # noqa: E731
    g, want, q = torch.Generator().manual_seed(3), [], c.q
    for r, (n, length) in enumerate(shape):
        if not n:
            continue
        lo, hi = seen(c, r, window)
        pick = torch.rand((n, heads), generator=g)
        pick[torch.rand((n, heads), generator=g) < 0.2] = 0.0  # the first and the last key that a row sees, more often
        pick[torch.rand((n, heads), generator=g) < 0.2] = 1.0
        j = (lo[:, None] + (pick * (hi - lo)[:, None]).long().clamp(max=(hi - lo - 1)[:, None])).cuda()
        page, off, head = c.table[r].long()[j // c.page], j % c.page, (torch.arange(heads, device="cuda") // (heads // kv)).expand(n, -1)
        q[sum(c.counts[:r]):sum(c.counts[:r + 1])] = wide(c.key[page, head, off]).half()
        want.append(wide(c.value[page, head, :, off]) * c.value_scale)
    want = torch.cat(want)
    # the key's score is 60, another one's at most about 30: a probability of 1, and below e^-25 for all others together
    got = c.run(pk, *window, scale=60 / (128 * c.key_scale))[:sum(c.counts)]
    plain.close(got, want, want.abs() * 2 * plain.U16 + plain.TINY16 + 6 * 2.0**-36)
