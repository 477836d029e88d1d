"""Attention of new tokens over the paged cache against its definition in 64 bits."""
import pytest

torch = pytest.importorskip("torch")

import serving_plain as plain  # noqa: E402
from test_gpu_parity import pk  # noqa: E402, F401

pytestmark = pytest.mark.gpu


def gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


class Case:
    """Sequences of (new tokens, keys) over a shuffled cache; every place that no key fills holds NaN."""

    wider = 0  # keys that the tables are wider than they need to be

    def __init__(self, shape, heads=4, kv=2, d=128, page=16, fp8=False, seed=1, spare_rows=3, peak=1.0):
        g = gen(seed)
        self.heads, self.kv, self.d, self.page, self.fp8 = heads, kv, d, page, fp8
        self.counts, self.lengths_ = [n for n, _ in shape], [length for _, length in shape]
        columns = max(max(-(-length // page) for length in self.lengths_), 1) + 1 + self.wider // page
        pages = sum(-(-length // page) for length in self.lengths_) + 3
        ids = torch.randperm(pages, generator=g, device="cuda").int()
        self.table = torch.full((len(shape), columns), 2 ** 30, dtype=torch.int32, device="cuda")  # never a page
        kind = torch.uint8 if fp8 else torch.float16
        nothing = 0x7F if fp8 else float("nan")
        self.key = torch.full((pages, kv, page, d), nothing, dtype=kind, device="cuda")
        self.value = torch.full((pages, kv, d, page), nothing, dtype=kind, device="cuda")
        self.key_scale, self.value_scale = (0.25, 0.5) if fp8 else (1.0, 1.0)
        at = 0
        for r, length in enumerate(self.lengths_):
            n = -(-length // page)
            self.table[r, :n] = ids[at:at + n]
            at += n
            k, v = (torch.randn((length, kv, d), generator=g, device="cuda") * x for x in (peak, 1.0))
            if fp8:
                k, v = ((x / s).to(torch.float8_e4m3fn).view(torch.uint8) for x, s in ((k, self.key_scale), (v, self.value_scale)))
            else:
                k, v = k.half(), v.half()
            plain.to_pages(k, v, page, self.table[r].long(), self.key, self.value)
        tokens = sum(self.counts)
        self.starts = torch.tensor([sum(self.counts[:i]) for i in range(len(shape) + 1)], dtype=torch.int32, device="cuda")
        self.lengths = torch.tensor(self.lengths_, dtype=torch.int32, device="cuda")
        wide = torch.randn((tokens + spare_rows, heads + kv, d), generator=g, device="cuda").half()
        self.q = wide[:, :heads]  # a slice of a projection's rows
        self.q[tokens:] = float("nan")
        self.out = torch.full((tokens + spare_rows, heads, d), 9.0, dtype=torch.float16, device="cuda")
        self.most = max(max(self.counts), 0)

    def workspace(self, pk):  # noqa: F811
        size = pk.paged_attention_workspace_bytes(self.q.shape[0], self.most, len(self.counts), self.heads, self.kv, self.d, self.page, self.table.shape[1])
        return torch.full((size,), 0xFF, dtype=torch.uint8, device="cuda")  # its content must not matter

    def run(self, pk, left=-1, right=0, scale=None, workspace=None, out=None, **kw):  # noqa: F811
        out = self.out if out is None else out
        pk.paged_attention(self.q, self.key, self.value, self.table, self.starts, self.lengths, out, self.workspace(pk) if workspace is None else workspace,
                           max_queries=kw.pop("max_queries", self.most), left=left, right=right, scale=scale, key_scale=self.key_scale,
                           value_scale=self.value_scale, **kw)
        return out

    def check(self, pk, left=-1, right=0, scale=None, **kw):  # noqa: F811
        got = self.run(pk, left, right, scale, **kw)
        tokens = sum(self.counts)
        want, bound = plain.attention(self.q[:tokens], self.key, self.value, self.table, self.starts, self.lengths, left, right,
                                      self.d ** -0.5 if scale is None else scale, self.key_scale, self.value_scale)
        plain.close(got[:tokens], want, bound, f"{self.counts} over {self.lengths_}, window ({left}, {right})")
        assert (got[tokens:] == 9).all()
        return got


@pytest.fixture(autouse=True, params=[0, 6000])
def tables(request):
    """Everything with tables as wide as the longest sequence, and with wide ones, whose keys are dealt in shares."""
    Case.wider = request.param
    yield
    Case.wider = 0


@pytest.mark.parametrize("length", [1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 200, 255, 256, 257, 511, 513, 1000, 2049, 5000])
@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("d", [64, 128])
def test_one_token(pk, length, fp8, d):  # noqa: F811
    Case([(1, length)], d=d, fp8=fp8, seed=length, page=(16, 64)[length % 2]).check(pk)


@pytest.mark.parametrize("heads,kv", [(1, 1), (8, 8), (8, 1), (12, 4), (16, 1), (17, 1), (20, 1), (40, 1), (6, 2), (35, 5), (64, 8)])
@pytest.mark.parametrize("fp8", [False, True])
def test_heads(pk, heads, kv, fp8):  # noqa: F811
    Case([(1, 77), (3, 150), (2, 2)], heads=heads, kv=kv, fp8=fp8, seed=heads).check(pk)


@pytest.mark.parametrize("page", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("left,right", [(-1, 0), (-1, -1), (20, 0), (0, 0), (128, 16), (40, -1), (5, 3)])
def test_windows_and_pages(pk, page, fp8, left, right):  # noqa: F811
    Case([(1, 300), (7, 7), (5, 333), (40, 90), (0, 50), (1, 1), (2, 700)], page=page, fp8=fp8, seed=page).check(pk, left, right)


@pytest.mark.parametrize("shape", [
    [(16, 16)], [(17, 40)], [(33, 33), (1, 900)], [(64, 64)], [(65, 1000)], [(100, 2000), (3, 5), (1, 4000)], [(130, 131)], [(200, 777), (129, 129)],
    [(0, 0), (5, 5), (0, 9), (0, 0)], [(300, 300)],
])
@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("heads,kv,d", [(4, 2, 128), (4, 4, 64), (10, 2, 128)])
def test_chunks(pk, shape, fp8, heads, kv, d):  # noqa: F811
    Case(shape, heads=heads, kv=kv, d=d, fp8=fp8, seed=len(shape), page=32).check(pk)


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("left,right", [(128, 0), (128, 16), (60, -1), (-1, -1), (0, 0)])
def test_chunk_windows(pk, fp8, left, right):  # noqa: F811
    Case([(150, 600), (70, 70), (90, 1300)], fp8=fp8, seed=6, page=64).check(pk, left, right)


@pytest.mark.parametrize("fp8", [False, True])
def test_ragged_batch(pk, fp8):  # noqa: F811
    Case([(1, 1 + 137 * i % 1900) for i in range(70)], heads=8, kv=2, fp8=fp8, page=32, seed=11).check(pk)


def test_many_short_sequences(pk):  # noqa: F811
    Case([(i % 3, 1 + 37 * i % 100 + i % 3) for i in range(600)], heads=2, kv=1, d=64, seed=12).check(pk)


def test_one_long_among_short(pk):  # noqa: F811
    Case([(1, 20), (1, 30000), (2, 10), (1, 64)], heads=8, kv=2, page=128, seed=13).check(pk)


@pytest.mark.parametrize("fp8", [False, True])
def test_rows_that_see_nothing_are_zero(pk, fp8):  # noqa: F811
    # more new tokens than keys: the first stand before key 0
    c = Case([(4, 9), (6, 6), (40, 40)], fp8=fp8, seed=14)
    c.lengths[1], c.lengths[2] = 2, 25
    got = c.check(pk)
    assert not got[4:8].any() and got[8:10].any() and not got[10:25].any() and got[25:50].any()
    c = Case([(3, 9), (2, 50)], fp8=fp8, seed=15)
    c.lengths[1] = 0
    got = c.check(pk)
    assert not got[3:5].any()
    assert not c.check(pk, -1, -1)[3:5].any()


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("left,right", [(-1, 0), (150, 20)])
def test_long_chunks_of_more_tokens_than_keys(pk, fp8, left, right):  # noqa: F811
    """Most row tiles see nothing, the last ones several tiles of keys."""
    c = Case([(1500, 1500), (3, 80), (900, 950)], fp8=fp8, seed=25, page=32)
    c.lengths[0], c.lengths[2] = 400, 700
    got = c.check(pk, left, right)
    assert not got[:1000].any() and got[1400:1500].any()


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("n", [6, 50])
def test_infinities_and_nan_in_unseen_keys(pk, fp8, n):  # noqa: F811
    """A later token's key and value are not seen by the earlier ones of the chunk, whatever they hold."""
    for place in ("key", "value"):
        for bad in ((0x7F,) if fp8 else (float("inf"), float("-inf"), float("nan"))):
            c = Case([(n, 100 + n)], fp8=fp8, seed=16)
            token = 100 + n - 3  # seen by the last three rows only
            p, off = int(c.table[0, token // 16]), token % 16
            if place == "key":
                c.key[p, :, off] = bad
            else:
                c.value[p, :, 5, off] = bad
            got = c.run(pk)
            assert torch.isfinite(got[:n - 3]).all(), (place, bad)
            want, bound = plain.attention(c.q[:n - 3], c.key, c.value, c.table, torch.tensor([0, n - 3]), c.lengths - 3, -1, 0, 128 ** -0.5, c.key_scale,
                                          c.value_scale)
            plain.close(got[:n - 3], want, bound, f"{place} {bad}")
            if place == "value":
                rows = got[n - 3:n].double()
                assert not torch.isfinite(rows[:, :, 5]).any() and torch.isfinite(rows[:, :, 6:]).all()
                if bad == float("inf"):
                    assert (rows[:, :, 5] == float("inf")).all()
            else:
                assert not torch.isfinite(got[n - 3:n]).any() or bad in (float("inf"), float("-inf"))


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("n", [1, 4, 60])
def test_pages_outside_the_cache_are_not_there(pk, fp8, n):  # noqa: F811
    c = Case([(n, 400 + n), (1, 33)], fp8=fp8, seed=17)
    c.table[0, 3], c.table[0, 9], c.table[1, 0] = -1, c.key.shape[0], -(2 ** 31)
    c.check(pk)


def test_lengths_beyond_the_table_are_cut(pk):  # noqa: F811
    c = Case([(1, 100), (2, 64)], seed=18, page=32)
    c.table = c.table[:, :4].contiguous()
    c.table[1] = c.table[0]
    c.lengths[1] = 2 ** 30  # 4 pages of 32 keys, the last partly NaN: only its first sequence's keys may be compared
    c.key[torch.isnan(c.key)], c.value[torch.isnan(c.value)] = 1.0, 1.0
    c.lengths_[1] = 128
    tokens = 3
    got = c.run(pk)
    lengths = torch.tensor([100, 128], dtype=torch.int32)
    want, bound = plain.attention(c.q[:tokens], c.key, c.value, c.table, c.starts, lengths, -1, 0, 128 ** -0.5)
    plain.close(got[:tokens], want, bound)


def test_shared_pages_and_batch_order(pk):  # noqa: F811
    """Two sequences with the same table and query give the same rows."""
    c = Case([(1, 500), (1, 500), (3, 40)], heads=8, kv=4, seed=19)
    c.table[1] = c.table[0]
    c.q[1] = c.q[0]
    got = c.check(pk)
    assert torch.equal(got[0], got[1]) or torch.allclose(got[0].float(), got[1].float(), rtol=2.0 ** -9, atol=2.0 ** -20)


@pytest.mark.parametrize("peak,scale", [(30.0, None), (1.0, 5.0), (0.0, None), (1.0, -0.3), (1.0, 0.0)])
def test_scores_large_small_and_equal(pk, peak, scale):  # noqa: F811
    Case([(1, 700), (30, 400)], peak=peak, seed=20).check(pk, scale=scale)


def test_a_slack_bound_on_queries(pk):  # noqa: F811
    """max_queries may be larger than any sequence's count."""
    c = Case([(1, 300), (2, 40), (1, 9)], heads=8, kv=2, seed=21, spare_rows=60)
    c.most = 64
    c.check(pk)


def test_output_as_a_slice(pk):  # noqa: F811
    c = Case([(3, 100), (1, 5)], seed=22)
    wide = torch.full((c.q.shape[0], 7, 128), 4.0, dtype=torch.float16, device="cuda")
    c.run(pk, out=wide[:, 2:6])
    want = c.check(pk)
    assert torch.equal(wide[:4, 2:6], want[:4]) and (wide[:, :2] == 4).all() and (wide[:, 6] == 4).all() and (wide[4:] == 4).all()


def test_one_token_whatever_its_stride(pk):  # noqa: F811
    """A single token's stride leads nowhere."""
    c = Case([(1, 100)], seed=26, spare_rows=0)
    wide = torch.zeros((1, 4 * 128 + 5), dtype=torch.float16, device="cuda")
    wide[:, :512] = c.q.reshape(1, 512)
    out = torch.full((1, 517), 4.0, dtype=torch.float16, device="cuda")
    c.q = wide[:, :512].unflatten(1, (4, 128))
    c.run(pk, out=out[:, :512].unflatten(1, (4, 128)))
    want = c.check(pk)
    assert torch.equal(out[:, :512], want.reshape(1, 512)) and (out[:, 512:] == 4).all()


def test_twice_the_same_bits(pk):  # noqa: F811
    c = Case([(1, 3000), (50, 800), (1, 40)], heads=8, kv=2, seed=23)
    first = c.run(pk).clone()
    for _ in range(3):
        assert torch.equal(c.run(pk), first)


def test_refusals_of_the_binding(pk):  # noqa: F811
    c = Case([(1, 50)], seed=24)
    ws = c.workspace(pk)
    with pytest.raises(ValueError):
        pk.paged_attention(c.q.float(), c.key, c.value, c.table, c.starts, c.lengths, c.out, ws, max_queries=1)
    with pytest.raises(ValueError):
        pk.paged_attention(c.q.transpose(1, 2), c.key, c.value, c.table, c.starts, c.lengths, c.out, ws, max_queries=1)
    with pytest.raises(ValueError):
        pk.paged_attention(c.q, c.key, c.value, c.table.long(), c.starts, c.lengths, c.out, ws, max_queries=1)
    with pytest.raises(ValueError):
        pk.paged_attention(c.q, c.key, c.value, c.table, c.starts[:1], c.lengths, c.out, ws, max_queries=1)
    with pytest.raises(ValueError):
        pk.paged_attention(c.q, c.key, c.key, c.table, c.starts, c.lengths, c.out, ws, max_queries=1)
    with pytest.raises(ValueError):
        pk.paged_attention(c.q.cpu(), c.key, c.value, c.table, c.starts, c.lengths, c.out, ws, max_queries=1)
    with pytest.raises(pk.PkError):
        pk.paged_attention(c.q, c.key, c.value, c.table, c.starts, c.lengths, c.out, ws, max_queries=10)
