"""GPU tests of block_matmul's larger tiles, each by the name of the kernel that the host chooses, against products in
float64 on the GPU.  Bounds are those of test_gpu_blocks; half of the cases have scales whose products lie beyond
float32, as in test_gpu_block_scales, and so results that f16 holds as subnormal numbers, 2^-24 apart, or not at all:
those are off by half of that, 2^-25, where half a step relative to the result is less."""

import numpy as np
import pytest

import block_ref as B
from pto_wsp import block_matmul
from pto_wsp._hip import NativeProgram
from pto_wsp.ir_bridge import workload_to_codegen_ir
from test_gpu_blocks import HALF, T, U, _dt, _torch, go

pytestmark = pytest.mark.gpu
TYPE = {"bf16": 0, "f16": 1, "f32": 2}


def number(codes, scale, rows):
    """Codes times their scales, in float64."""
    s = scale.double().repeat_interleave(128, 1)[:, :codes.shape[1]]
    return codes.double() * (s.repeat_interleave(128, 0)[:codes.shape[0]] if rows == 128 else s)


def eights(x):
    """[rows, columns / 8 (the last may be cut short), 8], as sizes."""
    torch = _torch()
    x = torch.nn.functional.pad(x.abs(), (0, -x.shape[1] % 8))
    return x.view(x.shape[0], -1, 8)


def most(x, y):
    """For each result the sum over eights of the largest of their terms' sizes."""
    torch = _torch()
    x, y, out = eights(x), eights(y), 0.0
    for k in range(x.shape[1]):
        terms = x[:, None, k, 0] * y[None, :, k, 0]
        for i in range(1, 8):
            terms = torch.maximum(terms, x[:, None, k, i] * y[None, :, k, i])
        out = out + terms
    return out


# Tile, whether rows go straight to LDS, type, M, N, K, scales beyond float32: K of one, two, three and more stages, whole
# and cut short, with shares of K; rows and columns that end inside a tile and at its end.
CASES = [
    ("256, 256", True, "bf16", 4300, 2304, 128, False), ("256, 256", True, "f16", 4300, 2304, 240, True), ("256, 256", True, "bf16", 4096, 2500, 272, True),
    ("256, 256", True, "f16", 4300, 2304, 640, False), ("256, 256", True, "bf16", 4096, 2304, 1024, True), ("256, 256", True, "bf16", 1300, 4096, 8192, False),
    ("128, 128", True, "bf16", 1000, 2600, 144, True), ("128, 128", True, "f16", 1024, 4096, 512, False), ("128, 128", True, "bf16", 1000, 2600, 1168, True),
    ("128, 128", True, "f32", 1900, 2500, 400, False), ("128, 128", True, "f32", 2048, 2560, 1024, True), ("128, 128", True, "bf16", 200, 2500, 8192, False),
    ("128, 128", False, "bf16", 1000, 2600, 333, True), ("128, 128", False, "f32", 1900, 2500, 515, False),
    ("64, 128", True, "bf16", 400, 4090, 400, True), ("64, 128", True, "f16", 400, 4096, 656, False), ("64, 128", False, "bf16", 400, 4090, 333, True),
    ("64, 64", True, "bf16", 230, 2500, 528, True), ("64, 64", False, "f16", 230, 2500, 333, False),
]


@pytest.mark.parametrize("tile,direct,dt,M,N,K,apart", CASES)
def test_tile(gpu, tile, direct, dt, M, N, K, apart):
    torch = _torch()
    rng = np.random.default_rng(M + N + K)
    t = {}
    for name, rows, block in (("a", M, 1), ("b", N, 128)):
        codes = torch.from_numpy(rng.integers(0, 256, size=(rows, K), dtype=np.uint8)).to(gpu)
        codes[(codes & 0x7F) == 0x7F] = 1
        t[name] = codes.view(torch.float8_e4m3fn)
        t[name + "_scale"] = torch.from_numpy(np.exp2(rng.normal(size=(-(-rows // block), B.blocks(K)))).astype(np.float32)).to(gpu)
    if apart:  # products of scales beyond float32 in a block of zeros, and 2^-110 of the others' in the next one
        t["a_scale"] *= 2.0 ** 90
        t["b_scale"] *= 2.0 ** -90
        t["a"].view(torch.uint8)[:, :128] &= 0x80
        t["b_scale"][:, 0] = 2.0 ** 100
        t["a_scale"][:, 1:2] *= 2.0 ** -110
    t["out"] = torch.full((M, N), float("nan"), dtype=_dt(dt), device=gpu)
    w = block_matmul(**{k: T(x) for k, x in t.items()})
    source = NativeProgram(workload_to_codegen_ir(w, "tile").module).precompile(0)
    assert f"BlockGemm<{tile}, " in source and f"{'true' if direct else 'false'}, {TYPE[dt]}>" in source
    go(w)
    x, y = number(t["a"], t["a_scale"], 1), number(t["b"], t["b_scale"], 128)
    want, size = x @ y.t().contiguous(), x.abs() @ y.abs().t().contiguous()
    bound = HALF[dt] * want.abs() + size * (2 * 128 + 4 + 2 * B.blocks(K)) * U + (2.0 ** -25 if dt == "f16" else 0.0)
    if dt != "f32":
        bound += 7 * 2.0 ** -13 * (1 + HALF[dt]) * most(x, y)
    top = torch.finfo(_dt(dt)).max
    got = t["out"].double()
    fine = want.abs() + bound <= top
    assert ((got - want).abs()[fine] <= bound[fine]).all() and fine.any()
    assert got[want.abs() - bound > top].isinf().all()
