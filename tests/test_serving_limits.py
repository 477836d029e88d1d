"""Sizes that the serving step's entry points refuse because a kernel could not answer them (no GPU is touched)."""
import pytest

from test_serving_refusals import ALIGN, ARG, P, SHAPE, status  # noqa: F401


@pytest.mark.parametrize("n,want", [(1 << 29, SHAPE), (1 << 30, SHAPE), ((1 << 29) - 1, ARG)])  # the last: only its missing output
def test_product_rows_of_one_launch(n, want):
    assert status("pk_gemv_int4g128", P, P, P, P, None, None, 1, 1, n, 128) == want
    assert status("pk_gemv_int4g128_a8", P, P, P, P, P, None, None, 1, 1, n, 128) == want
