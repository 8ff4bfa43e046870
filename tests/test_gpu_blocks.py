"""GPU tests of block_quantize, block_matmul and paged_norm_rotate, against plain forms in 64 bits (block_ref).

Codes are whole numbers and equal theirs, scales are float32 values and equal theirs.  With u = 2^-24, half a step
of float32, and half a step of the output's type (bf16 2^-8, f16 2^-11, f32 u):

* a product is off by half |out| + size * (2 * 128 + 4 + 2 * blocks) u, where size is the sum of its terms' sizes: a
  block's 128 products are exact and summed in float32, whose adders may cut instead of round (twice u each); their
  sum is multiplied with the product of two scales (u each) and added to the sums of the blocks before.  For 16-bit
  outputs the products are e4m3 MFMAs', which cut each of eight neighbouring products at 2^-13 of the largest: with
  1 at one place and 2^-k at another of the same eight, 2^-13 is in the sum and 2^-14 is not; at any place of another
  eight everything is, down to float32's last bit.  So seven of eight are off by less than 2^-13 of the largest each:
  7 * 2^-13 * the sum of the eights' largest terms (`most`) comes in addition.
* a rotated dim is off by half |out| + size * (D / 2 + 12) u, where size is |a c| + |b s|: the mean of D squares is
  off by (D + 3) u, half of that in its root, whose reciprocal, and the products with x and with the weight, take
  4 u; the rotation takes 3 u, and 2 u are for the terms of second order."""

import numpy as np
import pytest

import block_ref as B
import paged_ref as R
from pto_wsp import ExecutionError, block_matmul, block_quantize, paged_norm_rotate
from test_gpu_paged import HALF, T, _dt, _torch, go, ints

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


def f64(x):
    return x.detach().double().cpu().numpy()


def bits(codes):
    return codes.view(_torch().uint8).cpu().numpy()


def e4m3(gpu, codes):
    torch = _torch()
    return torch.from_numpy(np.ascontiguousarray(codes)).to(gpu).view(torch.float8_e4m3fn)


# ------------------------------------------------------------------------------ quantize
def check_quantize(x, rows, codes=None, scales=None):
    torch = _torch()
    M, K = x.shape
    codes = torch.full((M, K), 0.5, device=x.device).to(torch.float8_e4m3fn) if codes is None else codes
    scales = torch.full((-(-M // rows), B.blocks(K)), -1.0, device=x.device) if scales is None else scales
    go(block_quantize(x=T(x), codes=T(codes), scales=T(scales), rows=rows))
    want, s = B.quantize(f64(x), rows)
    assert np.array_equal(f64(scales), s)
    got = bits(codes)
    nan = (want & 0x7F) == 0x7F
    assert np.array_equal((got & 0x7F) == 0x7F, nan) and np.array_equal(got[~nan], want[~nan])


def numbers(gpu, M, K, dt, seed):
    torch = _torch()
    g = torch.Generator(device=gpu).manual_seed(seed)
    x = torch.randn((M, K), generator=g, device=gpu) * torch.exp2(3 * torch.randn((K,), generator=g, device=gpu))
    return x.to(_dt(dt))


@pytest.mark.parametrize("dt", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("rows", [1, 128])
@pytest.mark.parametrize("M,K", [(1, 1), (1, 128), (3, 127), (64, 256), (130, 129), (257, 1000), (5, 4096), (128, 136), (1100, 24)])
def test_quantize(gpu, M, K, rows, dt):
    check_quantize(numbers(gpu, M, K, dt, M + K), rows)


@pytest.mark.parametrize("rows", [1, 128])
def test_quantize_many(gpu, rows):
    check_quantize(numbers(gpu, 3000, 1152, "bf16", 1), rows)


@pytest.mark.parametrize("rows", [1, 128])
@pytest.mark.parametrize("dt", ["bf16", "f32"])
def test_quantize_strided(gpu, dt, rows):
    """Rows at odd distances and odd starts; what lies between the rows stays."""
    torch = _torch()
    buffer = numbers(gpu, 150, 333, dt, 2)
    codes = torch.full((150, 411), 1.0, device=gpu).to(torch.float8_e4m3fn)
    scales = torch.full((9, 150), -1.0, device=gpu)
    n = -(-150 // rows)
    check_quantize(buffer[:, 7:307], rows, codes[:, 5:305], scales.t()[:n, 2:5])
    assert (codes[:, :5].float() == 1).all() and (codes[:, 305:].float() == 1).all()
    assert (scales[:2] == -1).all() and (scales[5:] == -1).all()


@pytest.mark.parametrize("rows", [1, 128])
@pytest.mark.parametrize("dt", ["bf16", "f16", "f32"])
def test_quantize_values(gpu, dt, rows):
    """Zeros, infinities, NaN, the smallest and the largest numbers, and blocks of nothing else."""
    torch = _torch()
    x = numbers(gpu, 260, 400, dt, 3)
    info = torch.finfo(_dt(dt))
    x[0] = 0.0
    x[1] = info.smallest_normal / 4  # subnormal
    x[2] = info.max
    x[3, ::2], x[3, 1::2] = float("inf"), float("-inf")
    x[4] = float("nan")
    x[5, 3], x[5, 200], x[5, 399] = float("nan"), float("inf"), -info.max
    x[6, :128] = -0.0
    x[7] = info.smallest_normal
    x[130:] = 0.0
    x[200, 5] = float("-inf")
    check_quantize(x, rows)


# ------------------------------------------------------------------------------ matmul
def operands(gpu, M, N, K, seed):
    rng = np.random.default_rng(seed)
    a, b = (rng.integers(0, 256, size=s, dtype=np.uint8) for s in ((M, K), (N, K)))
    a[(a & 0x7F) == 0x7F] = 1
    b[(b & 0x7F) == 0x7F] = 2
    sa, sb = (np.exp2(rng.normal(size=s)).astype(np.float32) for s in ((M, B.blocks(K)), (B.blocks(N), B.blocks(K))))
    return a, sa, b, sb


def check_matmul(gpu, a, sa, b, sb, dt, lay=None):
    """lay: places for the operands and the result, by their names."""
    torch = _torch()
    put = {"a": e4m3(gpu, a), "a_scale": torch.from_numpy(sa).to(gpu), "b": e4m3(gpu, b), "b_scale": torch.from_numpy(sb).to(gpu)}
    t = {}
    for name, x in put.items():
        if lay and name in lay:
            lay[name].copy_(x) if x.dtype == torch.float32 else lay[name].view(torch.uint8).copy_(x.view(torch.uint8))
            x = lay[name]
        t[name] = x
    t["out"] = lay["out"] if lay and "out" in lay else torch.full((len(a), len(b)), float("nan"), dtype=_dt(dt), device=gpu)
    go(block_matmul(**{k: T(x) for k, x in t.items()}))
    want, size = B.matmul(a, sa, b, sb)
    got = f64(t["out"])
    bound = HALF[dt] * np.abs(want) + size * (2 * 128 + 4 + 2 * sa.shape[1]) * U
    if dt != "f32":
        bound = bound + 7 * 2.0 ** -13 * (1 + HALF[dt]) * B.most(a, sa, b, sb)
    over = np.abs(want) + bound > float(torch.finfo(_dt(dt)).max)  # in f16 what is off by so much may be infinite
    assert (np.abs(got - want)[~over] <= bound[~over]).all(), np.nanmax(np.abs(got - want)[~over] / bound[~over])
    assert np.isinf(got[(np.abs(want) - bound) > float(torch.finfo(_dt(dt)).max)]).all()
    return got


SHAPES = [(1, 1, 1), (1, 128, 128), (1, 4096, 1024), (2, 17, 16), (5, 1000, 1160), (16, 64, 128), (17, 130, 256), (33, 96, 200), (64, 1536, 512),
          (64, 256, 8192), (100, 127, 48), (128, 128, 128), (129, 257, 384), (200, 640, 144), (300, 1000, 1160), (256, 512, 640), (513, 768, 272),
          (1000, 512, 1024), (3, 5, 3000)]


@pytest.mark.parametrize("dt", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("M,N,K", SHAPES)
def test_matmul(gpu, M, N, K, dt):
    check_matmul(gpu, *operands(gpu, M, N, K, M + N + K), dt)


def test_matmul_large(gpu):
    """Against products in float64 on the GPU, of which the plain form has them."""
    torch = _torch()
    M, N, K = 2100, 2304, 2048
    a, sa, b, sb = operands(gpu, M, N, K, 4)
    t = {"a": e4m3(gpu, a), "a_scale": torch.from_numpy(sa).to(gpu), "b": e4m3(gpu, b), "b_scale": torch.from_numpy(sb).to(gpu)}
    out = torch.zeros((M, N), device=gpu)
    go(block_matmul(**{k: T(x) for k, x in t.items()}, out=T(out)))
    x = t["a"].double() * t["a_scale"].double().repeat_interleave(128, 1)
    y = t["b"].double() * t["b_scale"].double().repeat_interleave(128, 0).repeat_interleave(128, 1)
    want, size = x @ y.t().contiguous(), x.abs() @ y.abs().t().contiguous()
    assert ((out.double() - want).abs() <= want.abs() * U + size * (2 * 128 + 4 + 2 * 16) * U).all()


@pytest.mark.parametrize("M,N,K", [(37, 200, 272), (300, 384, 512), (6, 70, 100), (64, 512, 1024)])
@pytest.mark.parametrize("layout", ["padded", "odd", "transposed scales", "wide rows"])
def test_matmul_layouts(gpu, M, N, K, layout):
    """Rows that lie apart, at addresses that nothing divides; bytes between them are NaN codes, and what lies between the
    result's rows stays."""
    torch = _torch()
    a, sa, b, sb = operands(gpu, M, N, K, M)
    lay = {}
    gap, start = {"padded": (16, 16), "odd": (13, 3), "wide rows": (4096, 32)}.get(layout, (0, 0))
    if gap:
        for name, rows in (("a", M), ("b", N)):
            lay[name] = torch.full((rows * (K + gap) + 64,), 0x7F, dtype=torch.uint8, device=gpu).view(torch.float8_e4m3fn)[start:start + rows * (K + gap)].view(
                rows, K + gap)[:, :K]
        whole = torch.full((M, N + gap), 7.0, device=gpu)
        lay["out"] = whole[:, gap // 2:gap // 2 + N]
    else:
        lay["a_scale"] = torch.zeros((B.blocks(K), M), device=gpu).t()
        lay["b_scale"] = torch.zeros((B.blocks(K), B.blocks(N) + 1), device=gpu).t()[1:]
    check_matmul(gpu, a, sa, b, sb, "f32", lay)
    if gap:
        assert (whole[:, :gap // 2] == 7).all() and (whole[:, gap // 2 + N:] == 7).all()


@pytest.mark.parametrize("M,N,K", [(20, 256, 640), (300, 384, 640), (7, 33, 130)])
def test_matmul_not_finite(gpu, M, N, K):
    """A NaN code or scale reaches its own row or columns, an infinite scale makes infinities, zeros stay zeros."""
    torch = _torch()
    a, sa, b, sb = operands(gpu, M, N, K, 9)
    a[2, K - 1] = 0x7F
    b[5, 3] = 0xFF
    sa[4, 0] = np.nan
    sa[3, 1] = np.inf
    a[6] = 0
    out = torch.zeros((M, N), device=gpu)
    go(block_matmul(a=T(e4m3(gpu, a)), a_scale=T(torch.from_numpy(sa).to(gpu)), b=T(e4m3(gpu, b)), b_scale=T(torch.from_numpy(sb).to(gpu)), out=T(out)))
    got = f64(out)
    want, size = B.matmul(a, sa, b, sb)
    assert np.array_equal(np.isnan(got), np.isnan(want)) and np.array_equal(np.isinf(got), np.isinf(want))
    fine = np.isfinite(want)
    assert (np.abs(got - want)[fine] <= (np.abs(want) * U + size * (2 * 128 + 4 + 2 * sa.shape[1]) * U)[fine]).all()
    assert (got[6, [n for n in range(N) if n != 5]] == 0).all()


def test_matmul_twice_the_same(gpu):
    """Sums do not depend on which workgroup ends first."""
    torch = _torch()
    for M, N, K in ((1, 256, 16384), (64, 512, 8192), (160, 384, 4096)):
        a, sa, b, sb = operands(gpu, M, N, K, 10)
        outs = [check_matmul(gpu, a, sa, b, sb, "f32") for _ in range(3)]
        assert np.array_equal(outs[0], outs[1]) and np.array_equal(outs[0], outs[2])


# ------------------------------------------------------------------------------ norm and rotation
def rotate_case(gpu, counts, cached, Hq, Hk, D, R2, dt, seed, spare=2, offsets=False, weights=("q", "k"), wdt=None, positions=None):
    torch = _torch()
    g = torch.Generator(device=gpu).manual_seed(seed)
    counts, cached = np.asarray(counts), np.asarray(cached)
    starts = np.concatenate([[0], np.cumsum(counts)])
    rows = int(starts[-1]) + spare
    off = np.arange(len(counts)) * 3 if offsets else np.zeros(len(counts), int)
    most = positions or int((counts + cached + off).max()) + 1
    angles = np.outer(np.arange(most), 10000.0 ** (-np.arange(R2) / R2))
    t = {"q": torch.randn((rows, Hq, D), generator=g, device=gpu).to(_dt(dt)), "k": (3 * torch.randn((rows, Hk, D), generator=g, device=gpu)).to(_dt(dt)),
         "cos": torch.from_numpy(np.cos(angles).astype(np.float32)).to(gpu), "sin": torch.from_numpy(np.sin(angles).astype(np.float32)).to(gpu),
         "lengths": ints(gpu, counts + cached), "starts": ints(gpu, starts)}
    for x in "qk":
        t[x + "_out"] = torch.full_like(t[x], 9.0)
    for x in weights:
        t[x + "_weight"] = (1 + 0.3 * torch.randn((D,), generator=g, device=gpu)).to(_dt(wdt or dt))
    if offsets:
        t["offsets"] = ints(gpu, off)
    return t


def rotate_positions(t):
    starts, lengths = t["starts"].tolist(), t["lengths"].tolist()
    off = t["offsets"].tolist() if "offsets" in t else [0] * len(lengths)
    return np.array([off[b] + lengths[b] - (starts[b + 1] - r) for b in range(len(lengths)) for r in range(starts[b], starts[b + 1])], int)


def check_rotate(t, dt, eps=1e-6, interleaved=False, inputs=None):
    pos = rotate_positions(t)
    n = len(pos)
    for x in "qk":
        src = f64((inputs or t)[x])[:n]
        w = f64(t[x + "_weight"]) if x + "_weight" in t else None
        want, size = B.rotate(src, w, f64(t["cos"]), f64(t["sin"]), pos, eps, interleaved)
        got = f64(t[x + "_out"])
        bound = HALF[dt] * np.abs(want) + size * (src.shape[2] / 2 + 12) * U + (2.0 ** -25 if dt == "f16" else 0.0)  # f16: half its least step
        assert (np.abs(got[:n] - want) <= bound).all(), (x, np.max(np.abs(got[:n] - want) / bound))
        if inputs is None:
            assert (got[n:] == 9).all()


def rotate(t, **other):
    return paged_norm_rotate(**{k: T(x) for k, x in t.items()}, **other)


@pytest.mark.parametrize("dt", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("Hq,Hk,D,R2", [(4, 2, 128, 64), (32, 8, 128, 64), (7, 1, 80, 16), (5, 5, 96, 24), (3, 1, 16, 8), (2, 1, 256, 128), (9, 3, 64, 10),
                                        (1, 1, 192, 31), (2, 2, 256, 1), (3, 2, 176, 88), (1, 2, 48, 4)])
def test_rotate(gpu, Hq, Hk, D, R2, interleaved, dt):
    t = rotate_case(gpu, [3, 0, 1, 5], [10, 4, 0, 70], Hq, Hk, D, R2, dt, D + R2)
    go(rotate(t, interleaved=interleaved))
    check_rotate(t, dt, interleaved=interleaved)


@pytest.mark.parametrize("weights", [(), ("q",), ("k",)])
@pytest.mark.parametrize("D", [64, 80])
def test_rotate_weights(gpu, weights, D):
    """Heads without a weight are only rotated."""
    t = rotate_case(gpu, [1, 2], [3, 0], 6, 2, D, 8, "bf16", 1, weights=weights)
    go(rotate(t))
    check_rotate(t, "bf16")


@pytest.mark.parametrize("wdt", ["bf16", "f16", "f32"])
def test_rotate_weight_types_and_offsets(gpu, wdt):
    t = rotate_case(gpu, [4, 0, 2], [0, 9, 30], 4, 1, 128, 32, "f16", 2, offsets=True, wdt=wdt)
    go(rotate(t, eps=0.5))
    check_rotate(t, "f16", eps=0.5)


@pytest.mark.parametrize("batch", [1, 2, 63, 64, 65, 200, 4097])
def test_rotate_finds_its_request(gpu, batch):
    """Requests without rows among the others, at both ends too."""
    rng = np.random.default_rng(batch)
    counts = rng.integers(0, 3, size=batch)
    counts[[0, -1]] = 0
    counts[batch // 2] = 2
    t = rotate_case(gpu, counts, rng.integers(0, 50, size=batch), 2, 1, 64, 32, "f32", batch)
    go(rotate(t))
    check_rotate(t, "f32")


def test_rotate_many_rows(gpu):
    t = rotate_case(gpu, [3000, 1, 0, 2500], [5, 90, 2, 0], 12, 4, 128, 64, "bf16", 3)
    go(rotate(t))
    check_rotate(t, "bf16")


@pytest.mark.parametrize("dt", ["bf16", "f32"])
def test_rotate_in_place_and_packed(gpu, dt):
    """Queries, keys and values of a row in one buffer at an odd place, rotated where they lie; values stay."""
    torch = _torch()
    t = rotate_case(gpu, [3, 1, 40], [7, 0, 2], 6, 2, 80, 20, dt, 4)
    rows = len(t["q"])
    flat = torch.full((rows * 10 * 80 + 3,), 5.0, dtype=_dt(dt), device=gpu)
    packed = flat[3:].view(rows, 10, 80)
    packed[:, :6], packed[:, 6:8] = t["q"], t["k"]
    first = {"q": t["q"], "k": t["k"]}
    for x, at in (("q", packed[:, :6]), ("k", packed[:, 6:8])):
        t[x] = t[x + "_out"] = at
    for x in ("cos", "sin"):
        wide = torch.zeros((len(t[x]), 27), device=gpu)
        wide[:, 3:23] = t[x]
        t[x] = wide[:, 3:23]
    go(rotate(t))
    check_rotate(t, dt, inputs=first)
    assert (packed[:, 8:] == 5).all() and torch.equal(packed[-2:, :6], first["q"][-2:])


def test_rotate_values(gpu):
    """Zeros, large numbers, infinities and NaN stay within their heads."""
    torch = _torch()
    t = rotate_case(gpu, [6], [0], 3, 1, 64, 32, "f32", 5)
    t["q"][0, 0] = 0.0
    t["q"][1, 1] = 1e15
    t["q"][2, 0, 5], t["q"][3, 1, 60] = float("nan"), float("inf")
    go(rotate(t))
    got = f64(t["q_out"])
    assert (got[0, 0] == 0).all() and np.isfinite(got[[0, 1, 4, 5]]).all() and np.isnan(got[2, 0]).any()
    clean = torch.nan_to_num(t["q"], 0.0, 0.0, 0.0)
    want, size = B.rotate(f64(clean)[:6], f64(t["q_weight"]), f64(t["cos"]), f64(t["sin"]), rotate_positions(t), 1e-6, False)
    for r, h in ((0, 1), (1, 1), (2, 1), (2, 2), (3, 0), (4, 0)):
        assert (np.abs(got[r, h] - want[r, h]) <= size[r, h] * (64 / 2 + 13) * U).all()


@pytest.mark.parametrize("what", ["beyond", "negative", "starts"])
def test_rotate_out_of_range(gpu, what):
    """Rows whose position the tables lack raise and are left out, the others are written."""
    t = rotate_case(gpu, [2, 2], [3, 1], 2, 1, 64, 32, "f32", 6, positions=4 if what == "beyond" else None)
    if what == "negative":
        t["lengths"] = ints(gpu, [5, 1])
    if what == "starts":
        t["starts"] = ints(gpu, [0, 2, 2 + len(t["q"])])
    p = rotate(t).compile(target="hip_gfx950")
    p.execute()
    with pytest.raises(ExecutionError, match="paged_norm_rotate"):
        p.synchronize()
    got = f64(t["q_out"])
    left = {"beyond": [], "negative": [2], "starts": [2, 3]}[what]
    if what == "beyond":
        left = [r for r, p in enumerate(rotate_positions(t)) if p >= 4]
        assert left == [1]
    assert (got[left] == 9).all() and (got[0] != 9).all()
