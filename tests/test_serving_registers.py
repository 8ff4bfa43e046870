"""Kernels of the operators around paged_attention as a run builds them (on the CPU: launches are recorded instead
of run): no register is copied or spilled where only some lanes run, and none goes to scratch memory
(test_paged_registers has what happens where one does)."""

import glob

import pytest

import code_objects
import hip_stub
from pto_wsp import DType, block_matmul, block_quantize, paged_norm_rotate, paged_prefix_attention
from test_paged_host import T, cache

I32, F32, E4M3 = DType.I32, DType.F32, DType.F8E4M3
DT = {"bf16": DType.BF16, "f16": DType.F16, "f32": DType.F32, "e4m3": DType.F8E4M3, "i8": DType.I8}


def check(tmp_path, monkeypatch, workload, *names):
    monkeypatch.setenv("PTO_WSP_CODEGEN_CACHE_DIR", str(tmp_path))
    with hip_stub.program(workload) as once:
        entries = [x.entry for x in once()]
    assert set(names) <= set(entries)
    # None where another case of this process has built (and checked) the same kernels.
    for path in glob.glob(str(tmp_path / "hip" / "*.hsaco")):
        code = code_objects.kernels(path)
        bad = [(name, x) for name, instructions in code.items() for x in code_objects.ahead_of_restore(instructions)]
        assert not bad, "; ".join(f"{name}: {what}" for name, what in bad)
        spilled = {name: n for name, n in code_objects.scratch_bytes(path).items() if n}
        assert not spilled, spilled


@pytest.mark.parametrize("dt,code,H,D,page,G,rows,lse", [
    ("bf16", "e4m3", 8, 128, 16, 4, 64, False), ("bf16", "e4m3", 8, 128, 16, 4, 4096, True), ("f16", "i8", 2, 128, 8, 7, 64, True),
    ("f16", "e4m3", 8, 64, 32, 8, 2048, False), ("f32", "i8", 2, 80, 8, 7, 111, False), ("f32", "e4m3", 3, 256, 16, 4, 4096, True),
    ("bf16", "i8", 3, 240, 8, 7, 3, False), ("bf16", "i8", 3, 112, 24, 24, 900, True), ("f16", "i8", 3, 176, 64, 40, 2048, False),
    ("f32", "i8", 3, 144, 64, 5, 4096, False), ("bf16", "e4m3", 1, 96, 16, 24, 9000, True),
])
def test_prefix(tmp_path, monkeypatch, dt, code, H, D, page, G, rows, lse):
    other = {"lse": T(F32, rows, H * G)} if lse else {}
    check(tmp_path, monkeypatch, paged_prefix_attention(
        q=T(DT[dt], rows, H * G, D), out=T(DT[dt], rows, H * G, D), prefix_table=T(I32, 2, 9), prefix_lengths=T(I32, 2), members=T(I32, 3), page_table=T(I32, 40, 9),
        lengths=T(I32, 40), starts=T(I32, 41), **cache(DT[code], 100, H, page, D), **other), "ptowsp_paged_prefix_parts", "ptowsp_paged_prefix_merge")


@pytest.mark.parametrize("dt", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("K", [4096, 1160])
@pytest.mark.parametrize("M,N", [(1, 6144), (64, 6144), (300, 512), (300, 6144), (512, 6144), (8192, 6144)])
def test_matmul(tmp_path, monkeypatch, M, N, K, dt):
    kb = -(-K // 128)
    check(tmp_path, monkeypatch, block_matmul(a=T(E4M3, M, K), a_scale=T(F32, M, kb), b=T(E4M3, N, K), b_scale=T(F32, -(-N // 128), kb), out=T(DT[dt], M, N)),
          "ptowsp_block_matmul")


@pytest.mark.parametrize("dt", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("rows,M,K", [(1, 64, 4096), (1, 16384, 4096), (1, 16384, 1001), (128, 500, 300)])
def test_quantize(tmp_path, monkeypatch, rows, M, K, dt):
    check(tmp_path, monkeypatch, block_quantize(x=T(DT[dt], M, K), codes=T(E4M3, M, K), scales=T(F32, -(-M // rows), -(-K // 128)), rows=rows), "ptowsp_block_quantize")


@pytest.mark.parametrize("dt", ["bf16", "f32"])
@pytest.mark.parametrize("rows", [64, 16384])
@pytest.mark.parametrize("D,R,interleaved,weights", [(128, 128, False, "qk"), (80, 32, True, "q"), (256, 2, False, "qk"), (96, 50, True, ""), (192, 192, False, "k")])
def test_rotate(tmp_path, monkeypatch, D, R, interleaved, weights, rows, dt):
    w = {x + "_weight": T(DT[dt], D) for x in weights}
    check(tmp_path, monkeypatch, paged_norm_rotate(
        q=T(DT[dt], rows, 8, D), k=T(DT[dt], rows, 2, D), cos=T(F32, 99, R // 2), sin=T(F32, 99, R // 2), lengths=T(I32, 9), starts=T(I32, 10),
        q_out=T(DT[dt], rows, 8, D), k_out=T(DT[dt], rows, 2, D), interleaved=interleaved, **w), "ptowsp_paged_norm_rotate")
