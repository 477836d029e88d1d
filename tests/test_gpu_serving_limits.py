"""The serving step's operators at the largest sizes that they take."""
import pytest

torch = pytest.importorskip("torch")

from test_gpu_parity import pk  # noqa: E402, F401
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
