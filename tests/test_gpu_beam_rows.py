"""Rows of beams longer than a launch takes in one turn of its workgroups."""
import pytest

torch = pytest.importorskip("torch")

from test_gpu_parity import pk  # noqa: E402, F401

pytestmark = pytest.mark.gpu

# Out of place a launch has workgroups for 2^16 chunks of 512 units of 16 bytes a row, in place for 2^16 times 256 units.
TURN = (1 << 16) * 512 * 16


@pytest.mark.parametrize("row", [TURN - 1, TURN + 1, TURN + 16 * 512 * 3 + 5])
def test_rows_of_more_than_a_turn(pk, row):  # noqa: F811
    """Bytes that differ with their place and row, in both forms; odd lengths, so that the last unit overlaps the one before
    it out of place, and the last bytes are columns of their own in place."""
    beams = 3
    words = torch.arange(-(-beams * row // 4), dtype=torch.int32, device="cuda")
    words.mul_(-1640531535).bitwise_xor_(words >> 15).mul_(-2048144777)
    state = words.view(torch.uint8)[:beams * row].view(1, beams, row)
    del words
    parents = torch.tensor([[2, 0, 2]], dtype=torch.int32, device="cuda")
    out = torch.zeros_like(state)
    pk.beam_reorder(state, parents, out)
    for b, p in enumerate((2, 0, 2)):
        assert torch.equal(out[0, b], state[0, p])
    assert not torch.equal(state[0, 0], state[0, 2])
    pk.beam_reorder(state, parents, state)
    assert torch.equal(state, out)


def test_a_row_that_stays_within_a_long_state(pk):  # noqa: F811
    """A parent that is no row of the sequence leaves its row as it was, in every turn."""
    row = TURN + 16 * 512 * 2 + 7
    state = (torch.arange(2 * row, dtype=torch.int32, device="cuda") % 251).to(torch.uint8).view(1, 2, row)
    parents = torch.tensor([[-1, 0]], dtype=torch.int32, device="cuda")
    out = torch.full_like(state, 255)
    pk.beam_reorder(state, parents, out)
    assert bool((out[0, 0] == 255).all()) and torch.equal(out[0, 1], state[0, 0])
    first = state[0, 0].clone()
    pk.beam_reorder(state, parents, state)
    assert torch.equal(state[0, 0], first) and torch.equal(state[0, 1], first)
