"""Selection of beams over beams and vocabulary, and states that follow their beams."""
import math

import pytest

torch = pytest.importorskip("torch")

import decoding_plain as plain  # noqa: E402
from test_gpu_parity import pk  # noqa: E402, F401
from test_gpu_serving import gen  # noqa: E402

pytestmark = pytest.mark.gpu


class Search:
    def __init__(self, pk, n, beams, vocab, choices, fp16, seed=0, scale=3.0, flags=torch.bool):  # noqa: F811
        g = gen(seed + vocab + 13 * beams + choices)
        self.pk = pk
        self.logits = torch.randn((n, beams, vocab), generator=g, device="cuda") * scale
        if fp16:
            self.logits = self.logits.half()
        self.scores = -torch.rand((n, beams), generator=g, device="cuda") * 6
        self.ended, self.end, self.choices = None, -1, choices
        make = lambda kind, fill: torch.full((n, choices), fill, dtype=kind, device="cuda")  # noqa: E731
        self.out, self.tokens, self.parents, self.done = make(torch.float32, 7), make(torch.int32, -9), make(torch.int32, -9), make(flags, 1)
        self.workspace = torch.full((pk.beam_select_workspace_bytes(n, beams, vocab, choices),), 0xFF, dtype=torch.uint8, device="cuda")

    def run(self, stream=None):
        self.pk.beam_select(self.logits, self.scores, self.ended, self.out, self.tokens, self.parents, self.done, self.workspace, end_token=self.end,
                            stream=stream)

    def check(self):
        want = plain.select(self.logits.cpu(), self.scores.cpu(), None if self.ended is None else self.ended.cpu(), self.end, self.choices)
        assert self.tokens.tolist() == want[1]
        assert self.parents.tolist() == want[2]
        assert self.done.bool().tolist() == want[3]
        score = torch.tensor(want[0], dtype=torch.float64)
        got = self.out.double().cpu()
        assert torch.equal(torch.isinf(got), torch.isinf(score))
        real = ~torch.isinf(score)
        assert ((got - score).abs()[real] <= plain.U32 * (plain.SCORE_STEPS + score.abs()[real])).all()

    def go(self):
        self.run()
        self.check()


@pytest.mark.parametrize("n,beams,vocab,choices", [
    (1, 1, 1, 1), (3, 2, 2, 4), (2, 4, 5, 8), (1, 1, 63, 64), (2, 32, 7, 64), (4, 4, 1025, 4), (5, 3, 1030, 6), (1, 5, 16384, 5), (2, 2, 16385, 4),
    (1, 8, 16391, 16), (2, 3, 50021, 6), (1, 32, 40000, 64), (1, 1, 131071, 1), (1, 2, 1 << 20, 3), (70, 2, 100, 2)])
@pytest.mark.parametrize("fp16", [False, True])
def test_select(pk, n, beams, vocab, choices, fp16):  # noqa: F811
    Search(pk, n, beams, vocab, choices, fp16).go()


@pytest.mark.parametrize("vocab", [9, 1025, 40001])
@pytest.mark.parametrize("fp16", [False, True])
@pytest.mark.parametrize("flags", [torch.bool, torch.uint8])
def test_ended_and_dead_beams(pk, vocab, fp16, flags):  # noqa: F811
    s = Search(pk, 6, 4, vocab, 8, fp16, flags=flags)
    s.end = vocab // 2
    s.ended = torch.zeros(6, 4, dtype=flags, device="cuda")
    s.ended[0, 1] = s.ended[1] = s.ended[2, 3] = s.ended[5, 0] = 1
    s.scores[0, 0] = s.scores[4] = -math.inf
    s.scores[2, 3] = math.nan
    s.scores[3, 2] = math.inf
    s.scores[5] = torch.tensor([-1.0, -1.0, -1.0, -1.0])
    s.logits[0, 1] = math.nan  # not read
    s.logits[3, 0, s.end] = 40  # ends now
    s.go()
    assert s.parents[4].tolist() == [-1] * 8


@pytest.mark.parametrize("vocab", [33, 1025, 20000])
@pytest.mark.parametrize("fp16", [False, True])
def test_forbidden_tokens_nan_and_infinities(pk, vocab, fp16):  # noqa: F811
    s = Search(pk, 8, 2, vocab, 6, fp16)
    s.logits[0, 0] = -math.inf
    s.logits[1] = -math.inf
    s.logits[2, 0, 1:] = -math.inf
    s.logits[3, 0, vocab - 1] = math.nan
    s.logits[4, 1, 3] = math.inf
    s.logits[5, 0, : vocab - 2] = -math.inf
    s.logits[6] = -math.inf
    s.logits[6, 1, vocab - 1] = -60000.0
    s.logits[7, 0] = 65504.0 if fp16 else 3e38
    s.logits[7, 0, 5] = -65504.0 if fp16 else -3e38
    s.go()


@pytest.mark.parametrize("vocab", [2, 65, 1025, 16384, 30000])
@pytest.mark.parametrize("fp16", [False, True])
@pytest.mark.parametrize("choices", [3, 40])
def test_ties_go_to_the_lowest(pk, vocab, fp16, choices):  # noqa: F811
    s = Search(pk, 5, 4, vocab, choices, fp16)
    s.logits[0] = 1.5                      # all alike, in all beams
    s.logits[1, 1:] = s.logits[1, :1]      # equal rows
    s.logits[2] = s.logits[2].round()      # many alike
    s.logits[3] = s.logits[3].round() * 0  # zeros of both signs
    s.logits[4, :, : vocab // 2] = 2.0
    s.scores[0] = s.scores[1] = s.scores[3] = -2.0
    s.go()


@pytest.mark.parametrize("vocab", [33000, 131071])
@pytest.mark.parametrize("fp16", [False, True])
def test_equal_rows_at_all_alignments(pk, vocab, fp16):  # noqa: F811
    """Many wide rows (they are read in aligned blocks), each at another offset: equal ones tie, and a row's first and last
    logits and those at the borders of waves and parts are found at their places."""
    n, beams, per = 20, 16, 16 if fp16 else 8
    g = gen(vocab)
    row = torch.randn(vocab, generator=g, device="cuda")
    part = 2048 * (8 if fp16 else 4)
    spots = [0, 1, 7, 8, vocab - 1, vocab - 2, vocab - 9, 511, 512, 4095, 4096, part - 1, part, part + 1, 2 * part - 1]
    wide = torch.full((n, beams, vocab + 2 * per + 3), 30.0, device="cuda")
    for i in range(n):
        row2 = row.clone()
        row2[spots[i % len(spots)]] = 9.0
        wide[i, :, per:per + vocab] = row2
    wide = wide.half() if fp16 else wide
    s = Search(pk, n, beams, vocab, 20, fp16)  # strides are odd: every row lies at another alignment
    s.logits = wide[..., per:per + vocab]
    s.scores[:] = -1.0
    s.go()


def test_rows_a_stride_apart(pk):  # noqa: F811
    for fp16 in (False, True):
        s = Search(pk, 3, 4, 1031, 4, fp16)
        wide = torch.full((3, 4, 1100), 50.0, dtype=s.logits.dtype, device="cuda")
        wide[..., 7:1038] = s.logits
        s.logits = wide[..., 7:1038]
        s.go()


def test_beams_of_an_expanded_row_are_refused(pk):  # noqa: F811
    s = Search(pk, 2, 3, 100, 3, False)
    s.logits = torch.zeros(2, 1, 100, device="cuda").expand(2, 3, 100)
    with pytest.raises(ValueError):
        s.run()


@pytest.mark.parametrize("vocab", [1025, 33000])
def test_select_replays_and_workspaces(pk, vocab):  # noqa: F811
    """Replays over new values equal eager calls; a workspace for more serves fewer; two searches at once."""
    s = Search(pk, 4, 4, vocab, 4, True)
    s.workspace = torch.full((pk.beam_select_workspace_bytes(9, 8, 2 * vocab, 8),), 0xFF, dtype=torch.uint8, device="cuda")
    s.ended, s.end = torch.zeros(4, 4, dtype=torch.bool, device="cuda"), 3
    s.run()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        s.run()
    g = gen(3)
    for i in range(4):
        s.logits.copy_(torch.randn(s.logits.shape, generator=g, device="cuda") * 4)
        s.scores.copy_(-torch.rand((4, 4), generator=g, device="cuda") * 9)
        s.ended.copy_(torch.rand((4, 4), generator=g, device="cuda") < 0.3)
        s.workspace.fill_(i)
        graph.replay()
        torch.cuda.synchronize()
        s.check()
    sets = [Search(pk, 3, 4, vocab, 4, False, seed=k) for k in (5, 6)]
    streams = [torch.cuda.Stream() for _ in sets]
    torch.cuda.synchronize()
    for one, stream in zip(sets, streams):
        with torch.cuda.stream(stream):
            torch.cuda._sleep(200000)
        one.run(stream)
    torch.cuda.synchronize()
    for one in sets:
        one.check()


# ---- states ---------------------------------------------------------------------------

def reordered(state, parents, out):
    want = out.clone()
    n, beams = parents.shape
    for i in range(n):
        for b in range(beams):
            p = int(parents[i, b])
            if i * beams <= p < (i + 1) * beams:
                want[i, b] = state[i, p - i * beams]
    return want


@pytest.mark.parametrize("n,beams,row", [(1, 1, 1), (2, 3, 5), (8, 4, 2560), (3, 2, 1023), (1, 32, 4100), (5, 16, 640), (2, 8, 70000), (4, 5, 16), (300, 9, 7)])
@pytest.mark.parametrize("kind", [torch.float32, torch.float16, torch.uint8, torch.int64])
@pytest.mark.parametrize("in_place", [False, True])
def test_reorder(pk, n, beams, row, kind, in_place):  # noqa: F811
    g = gen(row)
    state = torch.randint(0, 100, (n, beams, row), generator=g, device="cuda").to(kind)
    parents = torch.randint(0, beams, (n, beams), generator=g, device="cuda") + beams * torch.arange(n, device="cuda")[:, None]
    odd = torch.rand((n, beams), generator=g, device="cuda")
    parents = torch.where(odd < 0.1, -1, torch.where(odd < 0.15, n * beams, torch.where(odd < 0.2, (parents + beams) % (n * beams), parents))).int()
    out = state if in_place else torch.full_like(state, 101)
    want = reordered(state, parents, out)
    pk.beam_reorder(state, parents, out)
    assert torch.equal(out, want)


@pytest.mark.parametrize("row", [1, 2, 255, 256, 257, 1023, 1024, 1028, 4080, 4096, 4112])
def test_reorder_of_short_rows(pk, row):  # noqa: F811
    """Rows of bytes at the border of the two ways, and parents that are no rows of their sequence."""
    g = gen(row)
    n, beams = 301, 6
    state = torch.randint(0, 256, (n, beams, row), generator=g, device="cuda", dtype=torch.uint8)
    parents = torch.randint(0, beams, (n, beams), generator=g, device="cuda") + beams * torch.arange(n, device="cuda")[:, None]
    wrong = torch.tensor([-1, -beams, -2**31, n * beams, 2**31 - 1, 0], device="cuda")[torch.randint(0, 6, (n, beams), generator=g, device="cuda")]
    parents = torch.where(torch.rand((n, beams), generator=g, device="cuda") < 0.3, wrong, parents).int()
    out = torch.randint(0, 256, (n, beams, row), generator=g, device="cuda", dtype=torch.uint8)
    want = reordered(state, parents, out)
    pk.beam_reorder(state, parents, out)
    assert torch.equal(out, want)


@pytest.mark.parametrize("shift", [1, 2, 4, 8])
def test_reorder_of_unaligned_states(pk, shift):  # noqa: F811
    whole = torch.randint(0, 256, (shift + 3 * 4 * 96 + 64,), device="cuda").to(torch.uint8)
    state = whole[shift:shift + 3 * 4 * 96].view(3, 4, 96)
    parents = torch.tensor([[3, 2, 1, 0], [4, 4, 4, 4], [11, 8, 9, 10]], dtype=torch.int32, device="cuda")
    before = whole.clone()
    want = reordered(state, parents, state)
    pk.beam_reorder(state, parents, state)
    assert torch.equal(state, want)
    assert torch.equal(whole[:shift], before[:shift]) and torch.equal(whole[shift + 3 * 4 * 96:], before[shift + 3 * 4 * 96:])


def test_reorder_of_many_chunks_a_row(pk):  # noqa: F811
    """More columns than one launch has workgroups for, in bytes and out of place."""
    row = (1 << 26) + 12345
    g = gen(9)
    state = torch.randint(0, 256, (1, 3, row), generator=g, device="cuda", dtype=torch.uint8)
    out = torch.zeros_like(state)
    parents = torch.tensor([[2, 0, 2]], dtype=torch.int32, device="cuda")
    pk.beam_reorder(state, parents, out)
    for b, p in enumerate((2, 0, 2)):
        assert torch.equal(out[0, b], state[0, p])
    before = state[0, :, :].clone()
    pk.beam_reorder(state, parents, state)
    for b, p in enumerate((2, 0, 2)):
        assert torch.equal(state[0, b], before[p])


def test_reorder_of_rows_of_more_than_32_bits(pk):  # noqa: F811
    row = (1 << 32) - 16
    state = torch.empty((1, 2, row // 8), dtype=torch.int64, device="cuda")
    state[0, 0], state[0, 1] = 5, 6
    state[0, 0, -1], state[0, 1, -1] = 7, 8
    pk.beam_reorder(state, torch.tensor([[1, 0]], dtype=torch.int32, device="cuda"), state)
    assert state[0, 0, 0] == 6 and state[0, 0, -1] == 8 and state[0, 1, 0] == 5 and state[0, 1, -1] == 7 and state[0, 0, row // 16] == 6


@pytest.mark.parametrize("n,beams,vocab", [(3, 4, 1025), (2, 8, 1027), (3, 16, 1030), (2, 16, 600), (2, 3, 30001), (1, 20, 9000), (2, 2, 70000)])
@pytest.mark.parametrize("choices", [16, 17, 32, 33, 64])
@pytest.mark.parametrize("fp16", [False, True])
def test_many_choices(pk, n, beams, vocab, choices, fp16):  # noqa: F811
    """Borders between the bounds of one wave and of all threads; then rows of which most is masked."""
    s = Search(pk, n, beams, vocab, choices, fp16, seed=5)
    s.go()
    g = gen(vocab)
    hidden = torch.rand(s.logits.shape, generator=g, device="cuda") < 0.97
    hidden[:, :, vocab // 3:] |= torch.rand((n, beams, 1), generator=g, device="cuda") < 0.5
    s.logits.masked_fill_(hidden, -math.inf)
    s.go()


@pytest.mark.parametrize("n,beams,vocab,choices", [(2, 4, 1025, 8), (2, 16, 1025, 4), (1, 2, 20000, 8), (1, 1, 70001, 64), (1, 20, 3000, 33)])
@pytest.mark.parametrize("fp16", [False, True])
def test_rows_masked_by_the_lowest_value(pk, n, beams, vocab, choices, fp16):  # noqa: F811
    """Fewer allowed tokens than choices: the rest are candidates all the same, the lowest indices first."""
    s = Search(pk, n, beams, vocab, choices, fp16, seed=9)
    allowed = torch.rand(s.logits.shape, generator=gen(choices), device="cuda") < 2.0 / vocab
    s.logits.masked_fill_(~allowed, torch.finfo(s.logits.dtype).min)
    if not fp16:
        s.scores[:, 1:] = -math.inf  # (scores near fp32's lowest value are all alike)
    s.go()
