"""GPU tests of block_matmul where the product of a row's scale and a column's lies beyond float32 though the results
do not: tolerances are those of test_gpu_blocks, whose terms hold here too.  A result's terms are sums of codes (2^-18
to 2^25 a block, or 0) times two scales; the sizes below keep the sums of the terms' sizes between 2^-114 and 2^127, so that what
float32 loses below 2^-126, half of 2^-149 for each block's sum, is less than 2^-15 of the bound."""

import numpy as np
import pytest

import block_ref as B
from pto_wsp import block_matmul
from test_gpu_blocks import T, _dt, _torch, check_matmul, e4m3, f64, go

pytestmark = pytest.mark.gpu
# The stream of up to 16 rows, small and larger tiles, rows at any address, shares of K.
SHAPES = [(5, 200, 1024), (16, 64, 128), (64, 512, 1024), (130, 1000, 1160), (300, 384, 512), (37, 70, 333), (1, 64, 16384), (160, 384, 4096)]


def operands(M, N, K, seed, low, high, ea, eb):
    """Codes of sizes between two of e4m3's bit patterns, scales around 2^ea and 2^eb."""
    rng = np.random.default_rng(seed)
    a, b = (rng.integers(low, high, size=s).astype(np.uint8) for s in ((M, K), (N, K)))
    sa, sb = (np.ldexp(1 + rng.random(s), e).astype(np.float32) for s, e in (((M, B.blocks(K)), ea), ((B.blocks(N), B.blocks(K)), eb)))
    return a, sa, b, sb


@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("ea,eb", [(-70, -66), (-126, -8), (-12, -122), (-3, -135), (-134, -4)])
@pytest.mark.parametrize("M,N,K", SHAPES)
def test_scales_whose_product_is_too_small(gpu, M, N, K, ea, eb, dt):
    """Codes of 128 and more: 2^14 and more for each column, times 2^-138."""
    check_matmul(gpu, *operands(M, N, K, M + N, 0x70, 0x7F, ea, eb), dt)


@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("ea,eb", [(64, 64), (119, 4), (2, 125), (9, 119), (127, -4), (-3, 127)])
@pytest.mark.parametrize("M,N,K", SHAPES)
def test_scales_whose_product_is_too_large(gpu, M, N, K, ea, eb, dt):
    """Codes of 2^-9 to 7 * 2^-9 (2 * 2^-9 in long rows), of either sign in a; rows and blocks of zeros among them, whose
    results are 0."""
    a, sa, b, sb = operands(M, N, K, M + N, 1, 8 if K < 2048 else 3, ea, eb)
    a ^= np.random.default_rng(1).integers(0, 2, size=a.shape).astype(np.uint8) << 7
    a[:, :128] = 0
    a[M // 2] = 0
    b[N // 2] = 0
    sa[:, 0] = 2.0 ** 120
    sb[:, 0] = 2.0 ** 120
    got = check_matmul(gpu, a, sa, b, sb, dt)
    assert (got[M // 2] == 0).all() and (got[:, N // 2] == 0).all()


@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("M,N,K", SHAPES)
def test_scales_at_the_ends(gpu, M, N, K, dt):
    """The least and the largest scales of float32 together, 0 and infinity: no result of zeros is NaN but those of 0
    times infinity, and blocks that are too small to matter add nothing."""
    torch = _torch()
    a, sa, b, sb = operands(M, N, K, M + N, 0x30, 0x7F, 0, 0)
    a[:, :128] = 0
    top, least = np.float32(np.finfo(np.float32).max), np.float32(2.0 ** -149)
    sa[:, 0], sb[:, 0] = top, top
    if B.blocks(K) > 1:
        sa[:, 1], sb[:, 1] = least, least
        sa[:M // 2, 1] = 0.0
    sa *= np.float32(2.0 ** -6)
    sa[:, 0] = top
    got = check_matmul(gpu, a, sa, b, sb, dt)
    assert np.isfinite(got).all() if dt != "f16" else not np.isnan(got).any()
    sa[M - 1, 0] = np.inf
    out = torch.zeros((M, N), dtype=_dt(dt), device=gpu)
    t = {"a": e4m3(gpu, a), "a_scale": torch.from_numpy(sa).to(gpu), "b": e4m3(gpu, b), "b_scale": torch.from_numpy(sb).to(gpu)}
    go(block_matmul(**{k: T(x) for k, x in t.items()}, out=T(out)))
    assert np.isnan(f64(out)[M - 1]).all() and np.array_equal(f64(out)[:M - 1], got[:M - 1])


@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("M,N,K", [(5, 200, 1024), (64, 512, 1024), (300, 384, 512), (37, 70, 333)])
def test_scales_of_any_sign_and_not_finite(gpu, M, N, K, dt):
    """Negative scales; infinite and NaN ones of weights reach their 128 columns, and no others."""
    torch = _torch()
    a, sa, b, sb = operands(M, N, K, M + N, 0x20, 0x70, 3, -3)
    rng = np.random.default_rng(2)
    sa, sb = (s * rng.choice(np.float32([-1, 1]), size=s.shape) for s in (sa, sb))
    got = check_matmul(gpu, a, sa, b, sb, dt)
    assert (got < 0).any() and (got > 0).any()
    sb[0, 1], sb[-1, 2] = np.inf, np.nan
    t = {"a": e4m3(gpu, a), "a_scale": torch.from_numpy(sa).to(gpu), "b": e4m3(gpu, b), "b_scale": torch.from_numpy(sb).to(gpu)}
    out = torch.zeros((M, N), dtype=_dt(dt), device=gpu)
    go(block_matmul(**{k: T(x) for k, x in t.items()}, out=T(out)))
    want = B.matmul(a, sa, b, sb)[0]
    now = f64(out)
    assert np.array_equal(np.isnan(now), np.isnan(want)) and np.array_equal(np.isinf(now), np.isinf(want))
    assert (np.sign(now) == np.sign(want))[np.isinf(want)].all()
    fine = np.isfinite(want)
    assert np.array_equal(now[fine], got[fine])
