"""Arguments that a scaling of rotary frequencies does not look at: whatever a caller has in them, the words are the same (no
GPU is touched)."""
import math

import pytest

pytest.importorskip("torch")

import parakeet_linear as pk

ODD = [0.0, -1.0, 1e300, math.inf, -math.inf, math.nan]


def words(scaling, factor=1.0, low=0.0, high=0.0, original=0, dim=64):
    return pk.rotary_frequencies(dim, 10000.0, scaling, factor, low, high, original, device="cpu").tolist()


@pytest.mark.parametrize("odd", ODD)
@pytest.mark.parametrize("dim", [16, 64, 256])
def test_plain(odd, dim):
    want = words(pk.ROTARY_PLAIN, dim=dim)
    assert abs(want[0] / 2**64 * 2 * math.pi - 1) <= 2.0**-46 and sorted(want, reverse=True) == want and min(want) > 0
    assert words(pk.ROTARY_PLAIN, odd, odd, odd, 2**31 - 1, dim) == want


@pytest.mark.parametrize("odd", ODD)
@pytest.mark.parametrize("name", ["LINEAR", "BASE"])
def test_borders_of_the_scalings_without_bands(name, odd):
    scaling = getattr(pk, "ROTARY_" + name)
    assert words(scaling, 8.0, odd, odd, 2**31 - 1) == words(scaling, 8.0)
