"""Builds libptowsp_hip.so in-tree (host library + embedded device templates).

The host side (IR parser, planner, cycle model, HIP emitter, hiprtc JIT and
the C ABI) is C++ compiled with hipcc; the device templates under
``csrc/device`` are embedded as strings and compiled per launch for gfx950
by hiprtc at run time.  ``check_device_templates()`` compiles a
representative kernel of every template family for gfx950 ahead of time,
which needs no GPU.
"""

import os
import subprocess
import sys

PKG_DIR = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(PKG_DIR)
CSRC = os.path.join(ROOT, "csrc")
INCLUDE = os.path.join(os.path.dirname(ROOT), "include")
BUILD_DIR = os.path.join(CSRC, "_build")
LIB_PATH = os.path.join(PKG_DIR, "libptowsp_hip.so")

HOST_SOURCES = ["module.cpp", "scalar.cpp", "analysis.cpp", "plan.cpp", "emit.cpp", "jit.cpp", "operators.cpp", "runtime.cpp", "noalloc.hip"]
DEVICE_HEADERS = [("kDeviceHeader", "ptowsp_device.h"), ("kLaunchHeader", "ptowsp_launch.h"), ("kPagedHeader", "ptowsp_paged.h"),
                  ("kPagedArgsHeader", "ptowsp_paged_args.h")]
DELIM = "PTOWSP_HDR"


def _write_embedded_headers() -> str:
    os.makedirs(BUILD_DIR, exist_ok=True)
    out = os.path.join(BUILD_DIR, "device_headers.inc")
    parts = ["// Generated by pto_wsp/_build.py from csrc/device/*.h; do not edit.\n"]
    for sym, name in DEVICE_HEADERS:
        with open(os.path.join(CSRC, "device", name), encoding="utf-8") as f:
            text = f.read()
        if f"){DELIM}\"" in text:
            raise RuntimeError(f"{name} contains the raw-string delimiter")
        parts.append(f'const char {sym}[] = R"{DELIM}({text}){DELIM}";\n')
    content = "".join(parts)
    old = open(out, encoding="utf-8").read() if os.path.exists(out) else None
    if old != content:
        with open(out, "w", encoding="utf-8") as f:
            f.write(content)
    return out


def build(verbose: bool = False) -> str:
    """Compile the host library with hipcc; returns the path of the .so."""
    _write_embedded_headers()
    srcs = [os.path.join(CSRC, "host", s) for s in HOST_SOURCES]
    tmp = LIB_PATH + ".tmp"
    cmd = [
        "hipcc", "-O2", "-std=c++17", "-fPIC", "-shared", "-Wall", "-Wextra",
        "--offload-arch=gfx950", "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
        "-I", INCLUDE, "-I", BUILD_DIR, "-I", os.path.join(CSRC, "host"),
        *srcs, "-o", tmp, "-lhiprtc",
    ]
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError("hipcc failed:\n" + " ".join(cmd) + "\n" + res.stdout + res.stderr)
    if verbose and (res.stdout or res.stderr):
        print(res.stdout + res.stderr, file=sys.stderr)
    os.replace(tmp, LIB_PATH)
    return LIB_PATH


def _operator_workloads():
    """The paged operators, in types and shapes that between them reach every kernel."""
    from pto_wsp import DType, Tensor, paged_attention, paged_plan, paged_store

    def T(dtype, *shape):
        return Tensor(data=None, shape=shape, dtype=dtype)

    i32, f32 = DType.I32, DType.F32
    yield paged_plan(lengths=T(i32, 4), counts=T(i32, 4), page_table=T(i32, 4, 8), free_pages=T(i32, 9), used=T(i32, 1),
                     new_lengths=T(i32, 4), new_used=T(i32, 1), starts=T(i32, 5), slots=T(i32, 7), page_size=16)
    bf16, f16, i8, e4m3 = DType.BF16, DType.F16, DType.I8, DType.F8E4M3
    for code, dt, heads, group, dim, page, rows, window in (
            # Few rows: 16 at a time and 32; prompts: tiles in bf16 and f16, rows one wave at a time.
            (e4m3, bf16, 8, 4, 128, 16, 4, 0), (i8, f16, 2, 7, 80, 8, 64, 9), (i8, f32, 1, 40, 256, 64, 4, 0), (e4m3, bf16, 1, 24, 128, 16, 4, 9),
            (e4m3, bf16, 8, 4, 128, 16, 1024, 0), (e4m3, f16, 2, 8, 64, 32, 1024, 9), (i8, bf16, 2, 4, 80, 24, 2048, 9), (i8, f32, 1, 40, 128, 16, 512, 0)):
        cache = {x + "_cache": T(code, 6, heads, page, dim) for x in "kv"} | {x + "_scale": T(f32, 6, heads) for x in "kv"}
        yield paged_store(k=T(dt, rows, heads, dim), v=T(dt, rows, heads, dim), slots=T(i32, rows), **cache)
        yield paged_attention(q=T(dt, rows, heads * group, dim), out=T(dt, rows, heads * group, dim), page_table=T(i32, 4, 3),
                              lengths=T(i32, 4), starts=T(i32, 5), window=window, lse=T(f32, rows, heads * group) if window else None, **cache)


def check_device_templates() -> None:
    """Build one kernel of each template family for gfx950 through hiprtc."""
    import numpy as np

    from pto_wsp import DType, Dense, In, InOut, Out, P, Tensor, Tile, kernel, pto, workload
    from pto_wsp._hip import NativeProgram

    f32, bf16 = DType.F32, DType.BF16
    x = Tensor(data=None, shape=(2, 4, 16, 128), dtype=f32)
    y = Tensor(data=None, shape=(2, 4, 16, 128), dtype=f32)

    @kernel
    def rmsnorm_tile(x: In[Tile[16, 128, f32]], out: Out[Tile[16, 128, f32]]):
        pto.store(out, pto.mul(x, pto.rsqrt(pto.rowmean(pto.mul(x, x)))))

    @kernel
    def softmax_tile(x: In[Tile[16, 128, f32]], out: Out[Tile[16, 128, f32]]):
        e = pto.exp(pto.sub(x, pto.rowmax(x)))
        pto.store(out, pto.div(e, pto.rowsum(e)))

    a = Tensor(data=None, shape=(2, 2, 2, 32, 16), dtype=bf16)
    b = Tensor(data=None, shape=(2, 2, 2, 16, 32), dtype=bf16)
    c = Tensor(data=None, shape=(2, 2, 2, 32, 32), dtype=f32)

    @kernel
    def gemm_tile(a_t: In[Tile[32, 16, bf16]], b_t: In[Tile[16, 32, bf16]], c_t: InOut[Tile[32, 32, f32]]):
        pto.store(c_t, pto.add(c_t, pto.matmul(a_t, b_t)))

    # MFMA GEMM family: 128x128 tasks, K step 64 (tile views [b][m][k] / [b][n][k] / [b][m][n]).
    ga = Tensor(data=None, shape=(1, 2, 2, 128, 64), dtype=bf16)
    gb = Tensor(data=None, shape=(1, 2, 2, 64, 128), dtype=bf16)
    gc = Tensor(data=None, shape=(1, 2, 2, 128, 128), dtype=f32)

    @kernel
    def mfma_tile(a_t: In[Tile[128, 64, bf16]], b_t: In[Tile[64, 128, bf16]], c_t: InOut[Tile[128, 128, f32]]):
        pto.store(c_t, pto.add(c_t, pto.matmul(a_t, b_t)))

    # Tile program with the PTO-ISA top-k ops (IOTA_U32, TSORT32, the index store).
    from pto_wsp import ptoisa, ptoisa_kernel

    sc = Tensor(data=None, shape=(2, 3, 1, 32), dtype=f32)
    ti = Tensor(data=None, shape=(2, 3, 1, 8), dtype=DType.I32)

    @ptoisa_kernel
    def topk8(scores: In[Tile[1, 32, f32]], out_idx: Out[Tile[1, 8, DType.I32]]):
        pairs = ptoisa.TSORT32(ptoisa.tload(scores), ptoisa.iota_u32(32))
        ptoisa.store_topk_indices_i32(out_idx, pairs, 8)

    @workload
    def wl():
        for i in P(Dense[1]()):
            for m in P(Dense[2]()):
                for n in P(Dense[2]()):
                    for k in P.seq(Dense[2]()):
                        mfma_tile[i, m, n, k](a_t=ga[i][m][k], b_t=gb[i][n][k], c_t=gc[i][m][n])
        for i in P(Dense[2]()):
            for t in P(Dense[4]()):
                rmsnorm_tile[i, t](x=x[i][t], out=y[i][t])
        for i in P(Dense[2]()):
            for t in P(Dense[4]()):
                softmax_tile[i, t](x=x[i][t], out=y[i][t])
        for i in P(Dense[2]()):
            for m in P(Dense[2]()):
                for k in P.seq(Dense[2]()):
                    gemm_tile[i, m, k](a_t=a[i][m][k], b_t=b[i][m][k], c_t=c[i][m][0])
        for i in P(Dense[2]()):
            for t in P(Dense[3]()):
                topk8[i, t](scores=sc[i][t], out_idx=ti[i][t])

    from pto_wsp.ir_bridge import workload_to_codegen_ir

    for w in _operator_workloads():
        NativeProgram(workload_to_codegen_ir(w, "operator_check").module).precompile(0)

    prog = NativeProgram(workload_to_codegen_ir(wl(), "template_check").module)
    for i in range(prog.num_launches()):
        prog.precompile(i)
    if "gemm program" not in prog.precompile(0, merged=True):
        raise RuntimeError("the MFMA GEMM template was not selected")
    if "ping-pong" not in prog.precompile(0, merged=True, pingpong=True):
        raise RuntimeError("the ping-pong GEMM template was not selected")
    del np


if __name__ == "__main__":
    print(build(verbose=True))
