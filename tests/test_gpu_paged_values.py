"""Paged attention over keys and values made so that each answer is known in closed form: probabilities far below the
largest one, infinities among them, scores of any size; and the same token in different company."""
import math

import pytest

torch = pytest.importorskip("torch")

import serving_plain as plain  # noqa: E402
from test_gpu_parity import pk  # noqa: E402, F401
from test_gpu_paged_attention import Case  # noqa: E402

pytestmark = pytest.mark.gpu

STEP = 32  # every 32nd key is a strong one: each wave and each part of the keys has some

# one launch; shares of several sequences' keys; chunks directly and in shares
SHAPES = [([(1, 700)], 0), ([(1, 700), (2, 300)], 6000), ([(1, 2500)] * 130, 0), ([(40, 500)], 0), ([(40, 3001), (77, 2000)] * 20, 6000)]


def put(c, key_or_value, r, token, feature, x, scale):
    """Feature `feature` of tokens `token` (a slice) of sequence r, all kv heads."""
    cache = c.key if key_or_value == "key" else c.value.transpose(2, 3)
    at = torch.arange(c.lengths_[r], device="cuda")[token]
    x = torch.tensor(x / scale, device="cuda")
    cache[c.table[r].long()[at // c.page], :, at % c.page, feature] = x.to(torch.float8_e4m3fn).view(torch.uint8) if c.fp8 else x.half()


def strong_and_weak(shape, wider, fp8, far):
    """Every STEP-th key has score `far` and value 1 in feature 1, the others score 0 and value 128 in feature 0; (case, scale)."""
    Case.wider = wider
    try:
        c = Case(shape, heads=2, kv=1, d=128, fp8=fp8, seed=5)
    finally:
        Case.wider = 0
    c.key.zero_()
    c.value.zero_()
    c.q.zero_()
    c.q[:, :, 0] = 8
    for r in range(len(shape)):
        put(c, "key", r, slice(0, None, STEP), 0, 8 * c.key_scale, c.key_scale)
        put(c, "value", r, slice(0, None), 0, 128.0, c.value_scale)
        put(c, "value", r, slice(0, None, STEP), 0, 0.0, c.value_scale)
        put(c, "value", r, slice(0, None, STEP), 1, 1.0, c.value_scale)
    return c, far / (64 * c.key_scale)


@pytest.mark.parametrize("shape,wider", SHAPES)
@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("far", [10.0, 14.5, 16.3, 17.6, 19.5])
def test_many_small_probabilities(pk, shape, wider, fp8, far):  # noqa: F811
    """Keys whose probability is e^-19 of the largest are not left out of the output, however many there are."""
    c, scale = strong_and_weak(shape, wider, fp8, far)
    got = c.run(pk, scale=scale).double().cpu()
    # two roundings to fp16 (probability and output); scores of up to 28 factors of two with four roundings; sums over at
    # most 64 products a step and, for these shapes, 200 steps, waves and parts, some of which truncate.  fp16 has no step
    # below 2^-24: next to a largest probability of 2^7 at least, each is also off by up to 2^-25 / 2^7 of that one, all
    # equal ones to the same side
    rel, each = 2 * plain.U16 + (4 * 28 + 2 * 264) * plain.U32, 2.0**-32
    for r, (n, length) in enumerate(shape):
        for i in range(n):
            seen = length - n + i + 1
            strong = -(-seen // STEP)
            weak = (seen - strong) * math.exp(-far)
            row = got[sum(c.counts[:r]) + i]
            for feature, want in ((0, 128 * weak / (strong + weak)), (1, strong / (strong + weak))):
                bound = want * rel + plain.TINY16 + 128 * (seen - strong) * each / (strong + weak)
                assert ((row[:, feature] - want).abs() <= bound).all(), (r, i, feature, row[:, feature], want, bound)
            assert not row[:, 2:].any()


@pytest.mark.parametrize("shape,wider", SHAPES)
@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("far", [3e5, 1e7, 1e9, 1e12, 1e20, -1e9])
def test_huge_scores(pk, shape, wider, fp8, far):  # noqa: F811
    """Scores whose fp32 steps are larger than 1: equal ones still share the sum equally, the others have none of it."""
    c, _ = strong_and_weak(shape, wider, fp8, 1.0)
    c.q[:, :, 0] = 7
    for r in range(len(shape)):
        put(c, "key", r, slice(0, None, STEP), 0, 9 * c.key_scale, c.key_scale)
    got = c.run(pk, scale=far / (63 * c.key_scale))[:sum(c.counts)]
    if far > 0:
        assert (got[:, :, 1] == 1).all() and not got[:, :, 0].any() and not got[:, :, 2:].any()
    else:  # the strong keys are the weak ones then; the first of a sequence's keys is a strong one
        alone = torch.tensor([length - n + i == 0 for n, length in shape for i in range(n)], device="cuda")
        assert not got[~alone][:, :, 1:].any() and (got[~alone][:, :, 0] == 128).all() and (got[alone][:, :, 1] == 1).all()


@pytest.mark.parametrize("shape,wider", SHAPES)
@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("far,lone", [(60.0, False), (300.0, False), (300.0, True)])
def test_infinity_of_a_tiny_probability(pk, shape, wider, fp8, far, lone):  # noqa: F811
    """A seen infinity (e4m3: NaN) reaches the rows that see it, the others not, however small its probability and wherever it
    stands; with a lone strong key the parts of the keys that do not hold it have a weight below fp32's smallest."""
    c, scale = strong_and_weak(shape, wider, fp8, far)
    if lone:
        for r in range(len(shape)):
            put(c, "key", r, slice(STEP, None, STEP), 0, 0.0, c.key_scale)
    clean = c.run(pk, scale=scale).clone()
    places = [(0, 5, 7, 1), (0, 131, 8, 2), (len(shape) - 1, 70, 9, 1), (len(shape) - 1, 201, 7, 2), (len(shape) // 2, shape[len(shape) // 2][1] - 2, 10, 1)]
    for r, token, feature, kind in places:
        p, off = int(c.table[r, token // c.page]), token % c.page
        c.value[p, :, feature, off] = 0x7F if fp8 else (0.0, float("inf"), float("-inf"))[kind]
    got = c.run(pk, scale=scale)
    want = clean.clone()
    for r, token, feature, kind in places:
        n, length = shape[r]
        first = max(0, token - (length - n))  # first row that sees it
        rows = want[sum(c.counts[:r]) + first:sum(c.counts[:r + 1])]
        rows[:, :, feature] += float("nan") if fp8 else (0.0, float("inf"), float("-inf"))[kind]  # both: NaN
    plain.close(got, want.double(), torch.zeros_like(want, dtype=torch.float64))


@pytest.mark.parametrize("left", [-1, 40, 130, 300])
@pytest.mark.parametrize("fp8", [False, True])
def test_a_row_in_other_company(pk, left, fp8):  # noqa: F811
    """In a table that takes one launch a token's bits are the same alone, behind others of its chunk, and among other sequences."""
    together = Case([(4, 420), (3, 700), (2, 5)], heads=8, kv=2, fp8=fp8, seed=9)
    got = together.run(pk, left=left)
    for r, (n, length) in enumerate([(4, 420), (3, 700), (2, 5)]):
        for i in range(n):
            at = sum(together.counts[:r]) + i
            q, out = together.q[at:at + 1].contiguous(), torch.empty((1, 8, 128), dtype=torch.float16, device="cuda")
            pk.paged_attention(q, together.key, together.value, together.table[r:r + 1], torch.tensor([0, 1], dtype=torch.int32, device="cuda"),
                               torch.tensor([length - n + i + 1], dtype=torch.int32, device="cuda"), out, None, max_queries=1, left=left,
                               key_scale=together.key_scale, value_scale=together.value_scale)
            assert torch.equal(out[0], got[at]), (r, i)


@pytest.mark.parametrize("shape,wider", SHAPES)
@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("far", [3e5, 1e7, 1e9, 1e12, 1e20, -1e9])
def test_huge_scores(pk, shape, wider, fp8, far):  # noqa: F811
    """Scores whose fp32 steps are larger than 1: equal ones still share the sum equally, the others have none of it."""
    c, _ = strong_and_weak(shape, wider, fp8, 1.0)
    c.q[:, :, 0] = 7
    for r in range(len(shape)):
        put(c, "key", r, slice(0, None, STEP), 0, 9 * c.key_scale, c.key_scale)
    got = c.run(pk, scale=far / (63 * c.key_scale))[:sum(c.counts)]
    if far > 0:
        assert (got[:, :, 1] == 1).all() and not got[:, :, 0].any() and not got[:, :, 2:].any()
    else:  # the strong keys are the weak ones then; the first of a sequence's keys is a strong one
        alone = torch.tensor([length - n + i == 0 for n, length in shape for i in range(n)], device="cuda")
        assert not got[~alone][:, :, 1:].any() and (got[~alone][:, :, 0] == 128).all() and (got[alone][:, :, 1] == 1).all()


@pytest.mark.parametrize("shape,wider", SHAPES)
def test_replays_over_changing_values(pk, shape, wider):  # noqa: F811
    """A replayed call over values that are finite, then infinite somewhere, then huge in their scores, then finite again equals
    the eager call each time."""
    c, _ = strong_and_weak(shape, wider, False, 60.0)
    ws, clean, query = c.workspace(pk), c.value.clone(), c.q.clone()
    scale = 60.0 / 64
    c.run(pk, scale=scale, workspace=ws)
    torch.cuda.synchronize()
    graph, out = torch.cuda.CUDAGraph(), torch.full_like(c.out, 7.0)
    with torch.cuda.graph(graph):
        c.run(pk, scale=scale, workspace=ws, out=out)
    for turn in range(5):
        c.value.copy_(clean)
        c.q.copy_(query * (1 if turn != 2 else 8000))
        if turn in (1, 3):
            for r in range(0, len(shape), 7):
                c.value[c.table[r, 5].long(), :, 40 + turn, 3] = float("inf")
        out.fill_(7.0)
        graph.replay()
        want = c.run(pk, scale=scale, out=torch.full_like(c.out, 7.0))
        assert torch.equal(out.isinf(), want.isinf()) and torch.equal(out.nan_to_num(), want.nan_to_num()) and not out.isnan().any()
        assert bool(out.isinf().any()) == (turn in (1, 3))
