"""Selection of beams some of which have no allowed token: rows of one finite value, whatever its size, are uniform."""
import math

import pytest

torch = pytest.importorskip("torch")

import decoding_plain as plain  # noqa: E402
from test_gpu_beams import Search  # noqa: E402
from test_gpu_parity import pk  # noqa: E402, F401

pytestmark = pytest.mark.gpu


def check(s):
    """Scores, tokens and parents from torch's log_softmax in 64 bits."""
    n, beams, vocab = s.logits.shape
    every = torch.log_softmax(s.logits.cpu().double(), 2) + s.scores.cpu().double()[:, :, None]
    best, at = torch.sort(every.view(n, beams * vocab), dim=1, descending=True, stable=True)
    best, at = best[:, :s.choices], at[:, :s.choices]
    got = s.out.cpu().double()
    assert ((got - best).abs() <= plain.U32 * (plain.SCORE_STEPS + best.abs())).all()
    assert torch.equal(s.tokens.cpu().long(), at % vocab)
    assert torch.equal(s.parents.cpu().long(), at // vocab + beams * torch.arange(n)[:, None])


# one launch of 4, 8 and 16 waves; two launches, of one and of several parts a row; bounds of one wave and of all threads
@pytest.mark.parametrize("n,beams,vocab,choices", [(3, 4, 1025, 4), (2, 7, 600, 40), (2, 16, 1025, 16), (2, 20, 700, 8), (2, 3, 20000, 8), (1, 2, 70001, 64)])
@pytest.mark.parametrize("value", ["lowest", -1e30, -6e4, 6e4, 1e17, 3e38])
@pytest.mark.parametrize("fp16", [False, True])
def test_a_beam_without_an_allowed_token_beside_live_ones(pk, n, beams, vocab, choices, value, fp16):  # noqa: F811
    s = Search(pk, n, beams, vocab, choices, fp16, seed=31)
    if value == "lowest":
        value = torch.finfo(s.logits.dtype).min
    elif abs(value) > 65504 and fp16:
        value = math.copysign(65504.0, value)
    s.logits[:, 0] = value
    s.logits[:, 1, 7] = 12.0
    s.scores[:] = -5.0
    s.run()
    check(s)
    assert (s.parents[:, 0] % beams != 0).all()  # any live beam's best token has more than a vocabulary's part
    s.scores[:, 1:] = -math.inf  # the masked beam alone: its first tokens, each with a vocabulary's part of its probability
    s.run()
    check(s)
    assert (s.parents % beams == 0).all() and s.tokens.tolist() == [list(range(choices))] * n


@pytest.mark.parametrize("vocab", [1025, 30001])
def test_few_of_the_largest_value(pk, vocab):  # noqa: F811
    """Of rows whose maxima are far from 0, what the maxima's number takes from their scores is kept."""
    s = Search(pk, 4, 3, vocab, 5, False, seed=32)
    for i, top in enumerate((1e8, 1e16, -1e25, 3e38)):
        for b, count in enumerate((1, 2, 40)):
            s.logits[i, b] = -3.4e38 if top < 0 else -top
            s.logits[i, b, 11:11 + count] = top
    s.scores[:] = torch.tensor([-2.0, -1.0, -0.5])
    s.run()
    check(s)


@pytest.mark.parametrize("beams", [2, 20])
def test_a_score_below_the_range_is_written_as_infinity(pk, beams):  # noqa: F811
    """Its token and parent are written all the same, in the order of the scores in 64 bits; as a beam it has no candidates then."""
    s = Search(pk, 1, beams, 9, 18, False, seed=33)
    s.scores[:] = -math.inf
    s.scores[0, 0], s.scores[0, 1] = -3e38, -1.0
    s.logits[0, 0] = -3e38
    s.logits[0, 0, 4] = 0.0
    s.logits[0, 1] = 1.0
    s.run()
    score = s.out.tolist()[0]
    assert score[:9] == [score[0]] * 9 and abs(score[0] + 1 + math.log(9)) < 1e-5 and score[9] == float(torch.tensor(-3e38))
    assert score[10:] == [-math.inf] * 8 and s.tokens.tolist()[0] == [*range(9), 4, 0, 1, 2, 3, 5, 6, 7, 8] and s.parents.tolist()[0] == [1] * 9 + [0] * 9
    s.scores[0, 1] = -math.inf
    s.scores[0, 0] = s.out[0, 12]
    s.run()
    assert s.tokens.tolist()[0] == [-1] * 18
