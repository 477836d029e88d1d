"""The serving step's operators at the largest sizes that they take."""
import pytest

torch = pytest.importorskip("torch")

from test_gpu_parity import pk  # noqa: E402, F401
from test_gpu_paged_attention import Case  # noqa: E402
from test_gpu_serving import randn, gen  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("int8", [False, True])
def test_norm_of_more_rows_than_a_launch_has_threads_for(pk, int8):  # noqa: F811
    """2^26 rows of 64 threads are 2^32: every row is written, and equals the same row of a short call."""
    g, rows, period = gen(1), (1 << 26) + 5, (1 << 16) + 3
    x, w = randn(g, period, 8), randn(g, 8)
    want, want_scales = torch.empty((period, 8), dtype=torch.int8 if int8 else torch.uint8, device="cuda"), torch.empty(period, device="cuda")
    want_h = torch.empty_like(x)
    pk.rms_norm_quantize(int(int8), x, x, w, want_h, want, want_scales, 1e-5)
    times = rows // period + 1
    many = x.repeat(times, 1)[:rows].contiguous()
    h, out, scales = torch.empty_like(many), torch.empty((rows, 8), dtype=want.dtype, device="cuda"), torch.full((rows,), -1.0, device="cuda")
    pk.rms_norm_quantize(int(int8), many, many, w, h, out, scales, 1e-5)
    assert torch.equal(scales, want_scales.repeat(times)[:rows])
    assert torch.equal(out, want.repeat(times, 1)[:rows]) and torch.equal(h, want_h.repeat(times, 1)[:rows])


def test_plan_of_the_most_slots(pk):  # noqa: F811
    """2^31 - 1 slots: those behind the last token are -1 up to the end, and nothing behind them is written."""
    capacity = 2**31 - 1
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    held, added, free, table = i32(5, 0, 20), i32(3, 0, 40), i32(*range(100, 110)), torch.full((3, 4), 7, dtype=torch.int32, device="cuda")
    starts, lengths, info = torch.empty(4, dtype=torch.int32, device="cuda"), torch.empty(3, dtype=torch.int32, device="cuda"), i32(9, 9, 9, 9)
    slots = torch.full((capacity + 1,), 5, dtype=torch.int32, device="cuda")
    pk.page_plan(held, added, free, i32(0, 10), table, starts, lengths, slots[:capacity], None, info, 16)
    assert info.tolist() == [43, 2, 0, 0] and lengths.tolist() == [8, 0, 60] and starts.tolist() == [0, 3, 3, 43]
    assert slots[:3].tolist() == [7 * 16 + 5, 7 * 16 + 6, 7 * 16 + 7] and slots[3:43].tolist() == [
        page * 16 + i for page, i in [(7, j) for j in range(4, 16)] + [(100, j) for j in range(16)] + [(101, j) for j in range(12)]]
    for part in slots[43:capacity].split(1 << 28):
        assert (part == -1).all()
    assert slots[capacity] == 5


@pytest.mark.parametrize("shape,wider", [([(1, 300), (4, 90)], 0), ([(1, 900), (2, 3000)], 6000), ([(40, 700), (90, 300)], 6000), ([(40, 400), (3, 3)], 0)])
@pytest.mark.parametrize("fp8", [False, True])
def test_attention_in_place_and_between(pk, shape, wider, fp8):  # noqa: F811
    """The output may take the queries' place, or lie between them in the same rows."""
    Case.wider = wider
    try:
        c = Case(shape, heads=4, kv=2, fp8=fp8, seed=41)
    finally:
        Case.wider = 0
    tokens = sum(c.counts)
    want = c.check(pk)[:tokens].clone()
    wide = torch.full((c.q.shape[0], 9, 128), 3.0, dtype=torch.float16, device="cuda")
    wide[:, 1:5] = c.q
    c.q = wide[:, 1:5]
    c.run(pk, out=wide[:, 5:])
    assert torch.equal(wide[:tokens, 5:], want) and (wide[tokens:, 5:] == 3).all() and (wide[:, 0] == 3).all()
    c.run(pk, out=c.q)
    assert torch.equal(wide[:tokens, 1:5], want) and torch.equal(wide[:tokens, 5:], want) and (wide[:, 0] == 3).all()


def test_integers_beyond_32_bits(pk):  # noqa: F811
    """No size and no window is cut to its low 32 bits."""
    big = 1 << 32
    c = Case([(3, 100), (1, 40)], seed=42)
    want, ws = c.run(pk).clone(), c.workspace(pk)
    for left, right in ((big + 5, 0), (-1, 0), (-big + 5, 0), (1 << 31, 0), ((1 << 31) - 1, 0)):
        assert torch.equal(c.run(pk, left=left, right=right, workspace=ws), want), (left, right)
    free = c.run(pk, left=-1, right=-1).clone()
    for right in (big, 1 << 31, -big, (1 << 31) - 1):
        assert torch.equal(c.run(pk, left=-1, right=right), free)
    with pytest.raises(ValueError):
        c.run(pk, max_queries=big + 3)
    with pytest.raises(ValueError):
        pk.paged_attention_workspace_bytes(big + 5, 5, 2, 16, 8, 128, 16, 400)
    with pytest.raises(pk.PkError):
        c.run(pk, max_queries=c.q.shape[0] + 1)  # more than there are
    wide = torch.empty((2, big + 8), dtype=torch.int32, device="cuda")
    with pytest.raises(ValueError):
        pk.paged_attention(c.q, c.key, c.value, wide, c.starts, c.lengths, c.out, ws, max_queries=3)
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    plan = lambda free, table, slots, page: pk.page_plan(i32(1, 2), i32(1, 1), free, i32(0, 4), table, i32(0, 0, 0), i32(0, 0), slots, None,  # noqa: E731
                                                         i32(0, 0, 0, 0), page)
    few, table = i32(1, 2, 3, 4), torch.zeros((2, 3), dtype=torch.int32, device="cuda")
    plan(few, table, i32(0, 0), 16)
    for bad in ((few, wide, i32(0, 0), 16), (few, table, wide.view(-1)[:big + 2], 16), (wide.view(-1)[:big + 2], table, i32(0, 0), 16),
                (few, table, i32(0, 0), big + 16)):
        with pytest.raises(ValueError):
            plan(*bad)
    del wide
    rows = torch.empty((big + 2, 8), dtype=torch.uint8, device="cuda")
    x = torch.empty((big + 2, 8), dtype=torch.float16, device="cuda")
    with pytest.raises(ValueError):
        pk.rms_norm_quantize(0, x, None, x[0], None, rows, torch.empty(big + 2, device="cuda"), 1e-5)
    del x, rows
    x, q = torch.empty((1, big + 128), dtype=torch.float16, device="cuda"), torch.empty((1, big // 8 + 16), dtype=torch.int32, device="cuda")
    s = torch.empty((1, big // 128 + 1), dtype=torch.float16, device="cuda")
    with pytest.raises(ValueError):
        pk.gemv_int4g128(x, q, s, s, None, torch.empty((1, 1), device="cuda"))


@pytest.mark.parametrize("heads,kv,shape", [(1024, 1, [(1, 100), (3, 50)]), (256, 256, [(1, 70), (2, 33)]), (1024, 256, [(2, 40)]), (1024, 64, [(1, 900)])])
@pytest.mark.parametrize("wider", [0, 6000])
def test_attention_of_the_most_heads(pk, heads, kv, shape, wider):  # noqa: F811
    Case.wider = wider
    try:
        Case(shape, heads=heads, kv=kv, d=64, seed=43).check(pk)
    finally:
        Case.wider = 0


@pytest.mark.parametrize("columns", [1, 40])
@pytest.mark.parametrize("n", [1, 256])
def test_attention_of_the_most_sequences_and_tokens(pk, columns, n):  # noqa: F811
    """4096 sequences, 2^20 tokens: with equal scores each row is the average of the keys it sees, all in the sequence's one page."""
    sequences, page, d = 4096, 256, 64
    tokens = sequences * n
    g = gen(44)
    key = torch.zeros((sequences, 1, page, d), dtype=torch.float16, device="cuda")
    value = torch.randint(-8, 9, (sequences, 1, d, page), generator=g, device="cuda").half()  # sums and their averages are exact in fp32
    ids = torch.randperm(sequences, generator=g, device="cuda")
    table = torch.full((sequences, columns), -1, dtype=torch.int32, device="cuda")
    table[:, 0] = ids
    lengths = torch.full((sequences,), page, dtype=torch.int32, device="cuda")
    if n == 1:
        lengths = torch.randint(1, page + 1, (sequences,), generator=g, device="cuda").int()
    starts = torch.arange(sequences + 1, device="cuda").int() * n
    q = randn(g, tokens, 1, d)
    out = torch.full_like(q, 9)
    size = pk.paged_attention_workspace_bytes(tokens, n, sequences, 1, 1, d, page, columns)
    pk.paged_attention(q, key, value, table, starts, lengths, out, torch.empty(size, dtype=torch.uint8, device="cuda"), max_queries=n)
    v = value[ids, 0].float().cumsum(2).transpose(1, 2)  # [sequence, keys, feature]
    seen = torch.arange(1, page + 1, device="cuda").float()
    want = v / seen[:, None] if n > 1 else (v / seen[:, None])[torch.arange(sequences, device="cuda"), lengths.long() - 1][:, None]
    # two roundings in fp32 and one to fp16
    off = (out.view(sequences, n, d).float() - want).abs() - want.abs() * (2.0**-11 + 2.0**-20) - 2.0**-24
    assert off.max() <= 0


def test_write_of_the_most_tokens(pk):  # noqa: F811
    tokens, page, d = 1 << 21, 128, 64
    g = gen(45)
    rows = randn(g, tokens, 2, d)
    pages = tokens // page
    ids = torch.randperm(pages, generator=g, device="cuda")
    slots = (ids[:, None] * page + torch.arange(page, device="cuda")).view(-1).int()
    key, value = torch.zeros((pages, 1, page, d), dtype=torch.float16, device="cuda"), torch.zeros((pages, 1, d, page), dtype=torch.float16, device="cuda")
    pk.paged_cache_write(rows[:, :1], rows[:, 1:], slots, key, value)
    assert torch.equal(key[ids, 0].view(tokens, d), rows[:, 0])
    assert torch.equal(value[ids, 0].transpose(1, 2).reshape(tokens, d), rows[:, 1])
