"""Host side of block_quantize, block_matmul, paged_norm_rotate and paged_prefix_attention, on the CPU: what compile()
refuses, and the launches of a run (recorded by hip_stub, so operands may be views of any size over a small buffer)."""

import re

import numpy as np
import pytest

import hip_stub
from pto_wsp import (CompileError, Dense, DType, P, block_matmul, block_quantize, paged_norm_rotate, paged_prefix_attention, sequential,
                     workload)
from pto_wsp._hip import NativeProgram
from pto_wsp.ir_bridge import workload_to_codegen_ir
from test_paged_host import T, cache

I32, F32, F16, BF16, E4M3, I8 = DType.I32, DType.F32, DType.F16, DType.BF16, DType.F8E4M3, DType.I8


def quantize(M=5, K=300, rows=1, dt=BF16, **other):
    return block_quantize(**dict(dict(x=T(dt, M, K), codes=T(E4M3, M, K), scales=T(F32, -(-M // rows) if rows > 0 else M, -(-K // 128)), rows=rows), **other))


def matmul(M=5, N=200, K=304, dt=BF16, **other):
    kb = -(-K // 128)
    return block_matmul(**dict(dict(a=T(E4M3, M, K), a_scale=T(F32, M, kb), b=T(E4M3, N, K), b_scale=T(F32, -(-N // 128), kb), out=T(dt, M, N)), **other))


def rotate(rows=5, Hq=4, Hk=2, D=64, R=32, batch=3, dt=BF16, **other):
    t = dict(q=T(dt, rows, Hq, D), k=T(dt, rows, Hk, D), cos=T(F32, 9, R // 2), sin=T(F32, 9, R // 2), lengths=T(I32, batch), starts=T(I32, batch + 1),
             q_out=T(dt, rows, Hq, D), k_out=T(dt, rows, Hk, D))
    return paged_norm_rotate(**dict(t, **other))


def prefix(rows=5, heads=2, G=4, D=64, batch=3, groups=2, dt=BF16, c=None, **other):
    t = dict(q=T(dt, rows, heads * G, D), out=T(dt, rows, heads * G, D), prefix_table=T(I32, groups, 7), prefix_lengths=T(I32, groups),
             members=T(I32, groups + 1), page_table=T(I32, batch, 4), lengths=T(I32, batch), starts=T(I32, batch + 1))
    return paged_prefix_attention(**dict(t | (c or cache(heads=heads, D=D)), **other))


@pytest.mark.parametrize("make,match", [
    (lambda: quantize(rows=2), "blocks of 2 rows"),
    (lambda: quantize(rows=-1), "blocks of -1 rows"),
    (lambda: quantize(K=0, scales=T(F32, 5, 0)), "x has no columns"),
    (lambda: quantize(codes=T(E4M3, 5, 301)), "codes has the shape"),
    (lambda: quantize(codes=T(I8, 5, 300)), "unsupported type i8"),
    (lambda: quantize(dt=I32), "unsupported type i32"),
    (lambda: quantize(scales=T(F32, 5, 2)), "scales has the shape"),
    (lambda: quantize(rows=128, scales=T(F32, 5, 3)), "scales has the shape"),
    (lambda: quantize(scales=T(BF16, 5, 3)), "unsupported type bf16"),
    (lambda: quantize(M=1 << 24, K=2048), "too many blocks"),
    (lambda: quantize(M=1, K=(1 << 30) + 1, rows=128), "too many blocks"),
    (lambda: quantize(x=T(BF16, 5, 300, 1)), "rank 2 is needed"),
    (lambda: matmul(b=T(E4M3, 200, 305)), "a has 304 columns, b 305"),
    (lambda: matmul(a=T(I8, 5, 304)), "unsupported type i8"),
    (lambda: matmul(N=0, b_scale=T(F32, 0, 3)), "b is empty"),
    (lambda: matmul(a_scale=T(F32, 5, 2)), "a_scale has the shape"),
    (lambda: matmul(b_scale=T(F32, 200, 3)), "b_scale has the shape"),
    (lambda: matmul(out=T(BF16, 200, 5)), "out has the shape"),
    (lambda: matmul(out=T(E4M3, 5, 200)), "unsupported type f8e4m3"),
    (lambda: rotate(k=T(BF16, 4, 2, 64)), "k has the shape"),
    (lambda: rotate(k=T(F16, 5, 2, 64), k_out=T(F16, 5, 2, 64)), "q and k differ in type"),
    (lambda: rotate(q_out=T(F32, 5, 4, 64)), "q and q_out differ in type"),
    (lambda: rotate(k_out=T(BF16, 5, 4, 64)), "k_out has the shape"),
    (lambda: rotate(D=72), "head size 72"),
    (lambda: rotate(D=272), "head size 272"),
    (lambda: rotate(R=66), "cos has the shape"),
    (lambda: rotate(sin=T(F32, 9, 8)), "sin has the shape"),
    (lambda: rotate(cos=T(BF16, 9, 16)), "unsupported type bf16"),
    (lambda: rotate(starts=T(I32, 3)), "starts has the shape"),
    (lambda: rotate(offsets=T(I32, 4)), "offsets has the shape"),
    (lambda: rotate(q_weight=T(BF16, 32)), "q_weight has the shape"),
    (lambda: rotate(q_weight=T(BF16, 64), k_weight=T(F32, 64)), "q_weight and k_weight differ in type"),
    (lambda: rotate(eps=-1.0), "eps"),
    (lambda: rotate(eps=float("nan")), "eps"),
    (lambda: prefix(members=T(I32, 2)), "members has the shape"),
    (lambda: prefix(prefix_lengths=T(I32, 3)), "prefix_lengths has the shape"),
    (lambda: prefix(prefix_table=T(I32, 2, 1 << 28)), "2\\^31 tokens"),
    (lambda: prefix(c=cache(D=32)), "q has the head size 64"),
    (lambda: prefix(c=cache(heads=3)), "8 query heads for 3 key heads"),
    (lambda: prefix(out=T(F32, 5, 8, 64)), "q and out differ in type"),
    (lambda: prefix(lse=T(F32, 5, 2)), "lse has the shape"),
    (lambda: prefix(starts=T(I32, 3)), "starts has the shape"),
    (lambda: prefix(page_table=T(I32, 2, 4)), "2 rows for 3 requests"),
    (lambda: prefix(scale=float("inf")), "scale"),
])
def test_refusals(make, match):
    with pytest.raises(CompileError, match=match):
        make().compile(target="hip_gfx950")


def test_operands_are_tensors():
    for make in (quantize, matmul, rotate, prefix):
        with pytest.raises(TypeError, match="must be a Tensor"):
            make(**{{quantize: "x", matmul: "a", rotate: "q", prefix: "q"}[make]: np.zeros(3)})


def entries(w):
    with hip_stub.program(w) as once:
        return [(x.entry.replace("ptowsp_", ""), x.blocks) for x in once()]


def test_empty_calls_launch_nothing():
    for w in (quantize(M=0), quantize(M=0, rows=128), matmul(M=0), rotate(rows=0), rotate(batch=0), prefix(rows=0), prefix(batch=0)):
        assert entries(w) == []


def test_launches():
    assert entries(quantize(64, 4096)) == [("block_quantize", 128)]
    assert entries(quantize(16384, 4096)) == [("block_quantize", 16384)]
    assert entries(quantize(300, 300, 128)) == [("block_quantize", 9)]
    assert [x for x, _ in entries(rotate())] == ["paged_norm_rotate"]
    # A line of tiles only where a group may have more than 64 rows a key head; prompts as in paged_attention.
    parts, units, finish, merge = "paged_prefix_parts", "paged_prefix_units", "paged_prefix_finish", "paged_prefix_merge"
    assert [x for x, _ in entries(prefix(rows=5))] == [parts, merge]
    assert [x for x, _ in entries(prefix(rows=40, batch=40))] == [parts, merge]
    assert [x for x, _ in entries(prefix(rows=1025))] == [units, parts, finish, merge]
    assert [x for x, _ in entries(prefix(rows=5, groups=0))] == [parts, merge]


@pytest.mark.parametrize("M,N,K,dt,tile,splits", [
    (1, 6144, 4096, BF16, "BlockStream<4, true, 0>", 1), (16, 256, 16384, BF16, "BlockStream<4, true, 0>", None), (64, 6144, 4096, BF16, "BlockGemm<32, 64, 1, 4, 6, true, 0>", 1),
    (128, 6144, 4096, F16, "BlockGemm<64, 64, 2, 2, 4, true, 1>", 1), (8192, 6144, 4096, BF16, "BlockGemm<256, 256, 4, 2, 2, true, 0>", 1),
    (8192, 6144, 4096, F32, "BlockGemm<128, 128, 2, 2, 4, true, 2>", 1), (300, 1000, 1160, F32, "false, 2>", None), (256, 4096, 14336, BF16, "BlockGemm<128, 128", None),
])
def test_tiles_of_a_product(M, N, K, dt, tile, splits):
    """The kernel that a build without a GPU makes is the one that a run launches; parts of K need a second launch."""
    prog = NativeProgram(workload_to_codegen_ir(matmul(M, N, K, dt), "build").module)
    source = prog.precompile(0)
    assert tile in source
    found = entries(matmul(M, N, K, dt))
    joined = len(found) == 2
    assert joined == ("ptowsp_block_matmul_join" in source) and len(found) <= 2
    if splits:
        assert joined == (splits > 1)
    if not joined and "BlockGemm" in source:
        bm, bn = map(int, re.search(r"BlockGemm<(\d+), (\d+),", source).groups())
        assert found == [("block_matmul", -(-M // bm) * -(-N // bn))]


def test_operands_at_execute():
    """Strides and overlaps, known when a run binds its tensors."""
    wide = T(BF16, 5, 300)
    wide.data = np.zeros((300, 5), np.uint16).T
    x = T(F32, 5, 300)
    out = T(BF16, 5, 200)
    out.data = np.zeros((200, 5), np.uint16).T
    q = T(BF16, 5, 4, 64)
    q.data = np.zeros((64, 4, 5), np.uint16).transpose(2, 1, 0)
    cos = T(F32, 9, 16)
    cos.data = np.zeros((16, 9), np.float32).T
    table = T(I32, 2, 7)
    table.data = np.zeros((7, 2), np.int32).T
    same = T(BF16, 5, 8, 64)
    scales = T(F32, 5, 3)
    scales.data = np.lib.stride_tricks.as_strided(np.zeros(9, np.float32), (5, 3), (0, 4))
    for w, match in ((quantize(x=wide), "x's last dimension must have stride 1"), (matmul(out=out), "out's last dimension must have stride 1"),
                     (quantize(scales=scales), "stride 0"), (rotate(q=q), "q's last dimension"), (rotate(cos=cos), "cos's last dimension"),
                     (prefix(prefix_table=table), "prefix_table's last dimension"), (prefix(q=same, out=same), "lies where q does"), (quantize(x=x, scales=x, K=300), None)):
        if match is None:
            with pytest.raises(CompileError):
                w.compile(target="hip_gfx950")
            continue
        with hip_stub.program(w) as once:
            with pytest.raises(RuntimeError, match=match):
                once()


def test_in_place():
    """Queries and keys are rotated where they lie, with the same strides; not upon each other."""
    q, k = T(BF16, 5, 4, 64), T(BF16, 5, 2, 64)
    assert len(entries(rotate(q=q, q_out=q, k=k, k_out=k))) == 1
    k_out = T(BF16, 5, 2, 64)
    k_out.data = q.data[:, :2]
    q_out = T(BF16, 5, 4, 64)
    q_out.data = q.data
    with hip_stub.program(rotate(q=q, q_out=q_out, k=k, k_out=k_out)) as once:
        with pytest.raises(RuntimeError, match="k_out"):
            once()


def test_captured_runs_keep_their_workspace():
    with hip_stub.program(sequential(matmul(256, 4096, 14336), prefix(rows=1025))) as once:
        with pytest.raises(RuntimeError):  # nothing has been allocated yet
            once(capture=True)
        n = len(once())
        assert n == 6 and len(once(capture=True)) == n
        with pytest.raises(RuntimeError, match="captured after a run"):
            once(capture=True)
        once()
        once(capture=True)


def test_loops_over_layers():
    """Operands indexed by a loop around the operators."""
    x, codes, scales = T(BF16, 3, 5, 256), T(E4M3, 3, 5, 256), T(F32, 3, 5, 2)
    b, bs, out = T(E4M3, 3, 128, 256), T(F32, 3, 1, 2), T(BF16, 3, 5, 128)

    @workload
    def wl():
        for layer in P.seq(Dense[3](), name="layer"):
            block_quantize(x=x[layer], codes=codes[layer], scales=scales[layer])
            block_matmul(a=codes[layer], a_scale=scales[layer], b=b[layer], b_scale=bs[layer], out=out[layer])

    assert [e for e, _ in entries(wl())] == ["block_quantize", "block_matmul"] * 3
