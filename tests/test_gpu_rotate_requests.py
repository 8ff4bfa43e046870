"""GPU tests of what paged_norm_rotate makes of requests' starts and lengths; tolerances are those of test_gpu_blocks."""

import numpy as np
import pytest

from pto_wsp import ExecutionError
from test_gpu_blocks import check_rotate, f64, go, ints, rotate, rotate_case

pytestmark = pytest.mark.gpu


def raises(t):
    p = rotate(t).compile(target="hip_gfx950")
    p.execute()
    with pytest.raises(ExecutionError, match="paged_norm_rotate"):
        p.synchronize()


@pytest.mark.parametrize("D", [64, 80])
def test_places_ahead_of_a_request(gpu, D):
    """A request of 1 token with 3 rows: the first two are none of its tokens, whatever its offset; they are left out."""
    t = rotate_case(gpu, [2, 3, 2], [3, 0, 4], 2, 1, D, 16, "f32", 1, offsets=True, positions=40)
    t["lengths"] = ints(gpu, [5, 1, 6])
    t["offsets"] = ints(gpu, [0, 16, 7])
    raises(t)
    got = f64(t["q_out"])
    assert (got[2:4] == 9).all() and (got[4] != 9).all()
    t["lengths"] = ints(gpu, [5, 3, 6])
    go(rotate(t))
    check_rotate(t, "f32")


@pytest.mark.parametrize("batch,where", [(4, 2), (3, 2), (64, 40), (65, 63), (300, 130), (5000, 4500)])
@pytest.mark.parametrize("what", ["down", "beyond", "below"])
def test_starts_out_of_order(gpu, batch, where, what):
    """One start that goes down, lies beyond the rows or below 0, behind any number of others; fewer waves than requests
    have 64 among them, too."""
    counts = np.zeros(batch, int)
    counts[[0, -1]] = 2, 1
    t = rotate_case(gpu, counts, np.full(batch, 3), 2, 1, 64, 16, "f32", batch, spare=1)
    t["starts"][where] = {"down": 1 if where < batch - 1 else 0, "beyond": len(t["q"]) + 1, "below": -1}[what]
    raises(t)


@pytest.mark.parametrize("batch", [64, 129, 5000])
def test_starts_beyond_the_rows(gpu, batch):
    """All rows are of requests in order; one behind them has rows that there are none of."""
    counts = np.zeros(batch, int)
    counts[3] = 4
    t = rotate_case(gpu, counts, np.full(batch, 3), 2, 1, 64, 16, "f32", batch, spare=0)
    go(rotate(t))
    check_rotate(t, "f32")
    t["starts"][-1] += 1
    raises(t)
