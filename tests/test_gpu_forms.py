"""Sizes at which the calls around a decoding step's cache go from one form of a kernel to another: both sides, against the
plain forms."""
import random

import pytest

torch = pytest.importorskip("torch")

from test_gpu_pages import Pool  # noqa: E402
from test_gpu_parity import pk  # noqa: E402, F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows,columns,spare", [
    (127, 20, 40), (128, 20, 40), (129, 20, 40), (128, 128, 40), (128, 129, 40), (113, 145, 40), (8, 60, (1 << 17) - 480), (8, 60, (1 << 17) - 479),
    (1024, 16, 40)])
def test_fork_in_one_launch_and_in_several(pk, rows, columns, spare):  # noqa: F811
    rng = random.Random(rows + columns)
    pool = Pool(rng, rows, columns, 16, spare=spare)
    for chance in (0.0, 0.1, 0.6):
        parents = [-1 if rng.random() < chance else min(rows - 1, r // 4 * 4 + rng.randrange(4)) for r in range(rows)]
        pool.go(pk, parents)
        pool.go(pk, parents, [int(rng.random() < 0.3) for _ in range(pool.pages)])
