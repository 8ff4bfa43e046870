"""GPU tests of paged_norm_rotate where a wave goes on with a token's next heads, several times: two waves a token, of
more than 32768 that its heads would take at once.  Against float64 on the GPU, by the bounds of test_gpu_blocks."""

import pytest

from test_gpu_blocks import HALF, U, _torch, go, rotate, rotate_case, rotate_positions

pytestmark = pytest.mark.gpu


def check(t, dt, interleaved):
    torch = _torch()
    pos = torch.from_numpy(rotate_positions(t)).to(t["q"].device)
    n, r = len(pos), t["cos"].shape[1]
    c, s = t["cos"].double()[pos][:, None], t["sin"].double()[pos][:, None]
    lo, hi = (slice(0, 2 * r, 2), slice(1, 2 * r, 2)) if interleaved else (slice(0, r), slice(r, 2 * r))
    for x in "qk":
        y = t[x][:n].double()
        if x + "_weight" in t:
            y = y / torch.sqrt((y * y).mean(-1, keepdim=True) + 1e-6) * t[x + "_weight"].double()
        want, size = y.clone(), y.abs()
        a, b = y[..., lo], y[..., hi]
        want[..., lo], want[..., hi] = a * c - b * s, b * c + a * s
        size[..., lo], size[..., hi] = (a * c).abs() + (b * s).abs(), (b * c).abs() + (a * s).abs()
        bound = HALF[dt] * want.abs() + size * (y.shape[2] / 2 + 12) * U + (2.0 ** -25 if dt == "f16" else 0.0)
        got = t[x + "_out"].double()
        assert ((got[:n] - want).abs() <= bound).all() and (got[n:] == 9).all()


@pytest.mark.parametrize("dt,Hq,Hk,D,R2,interleaved,weights", [
    ("bf16", 32, 8, 128, 64, False, ("q", "k")), ("f32", 29, 8, 128, 64, True, ("q",)), ("f16", 30, 10, 16, 1, False, ("q", "k")),
    ("bf16", 33, 7, 80, 16, False, ("k",)),
])
def test_turns(gpu, dt, Hq, Hk, D, R2, interleaved, weights):
    t = rotate_case(gpu, [5000, 1, 0, 2200], [5, 90, 2, 0], Hq, Hk, D, R2, dt, D, weights=weights)
    go(rotate(t, interleaved=interleaved))
    check(t, dt, interleaved)
