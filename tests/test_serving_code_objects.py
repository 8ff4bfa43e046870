"""Code objects of the operators around paged_attention, each built in a process of its own, where no test has built
(and kept) its kernels before: no register is copied or spilled where only some lanes run, none goes to scratch memory,
and no matrix instruction takes the powers of its codes from scalar registers, which it does not read."""

import json
import os
import re
import subprocess
import sys
import tempfile

import pytest

# Tile and threads, sizes, type.
MATMUL = [(256, 256, 512, 8192, 6144, 4096, "bf16"), (256, 256, 512, 4300, 2304, 640, "f16"), (128, 128, 256, 512, 6144, 4096, "bf16"),
          (128, 128, 256, 8192, 6144, 4096, "f32"), (128, 128, 256, 1000, 2600, 333, "bf16"), (128, 128, 256, 1900, 2500, 515, "f32"),
          (64, 128, 256, 400, 4090, 400, "bf16"), (64, 64, 256, 230, 2500, 528, "bf16"), (32, 64, 256, 64, 6144, 4096, "bf16"), (16, 16, 256, 16, 6144, 4096, "bf16"),
          (16, 16, 256, 5, 200, 1001, "f32")]
QUANTIZE = [(1, 64, 4096, "bf16"), (1, 16384, 1001, "f32"), (128, 500, 300, "f16")]
ROTATE = [("bf16", 16384, 128, 128, "qk"), ("f32", 64, 80, 32, "q"), ("bf16", 64, 256, 2, "")]
PREFIX = [("bf16", "e4m3", 8, 128, 16, 4, 64), ("bf16", "e4m3", 8, 128, 16, 4, 4096), ("f32", "i8", 2, 80, 8, 7, 111)]
CASES = [("matmul", *x) for x in MATMUL] + [("quantize", *x) for x in QUANTIZE] + [("rotate", *x) for x in ROTATE] + [("prefix", *x) for x in PREFIX]


def workload_of(case):
    from pto_wsp import DType, block_matmul, block_quantize, paged_norm_rotate, paged_prefix_attention
    from test_paged_host import T, cache

    I32, F32, E4M3 = DType.I32, DType.F32, DType.F8E4M3
    dts = {"bf16": DType.BF16, "f16": DType.F16, "f32": DType.F32, "e4m3": E4M3, "i8": DType.I8}
    op, *a = case
    if op == "matmul":
        _, _, _, M, N, K, dt = a
        kb = -(-K // 128)
        return block_matmul(a=T(E4M3, M, K), a_scale=T(F32, M, kb), b=T(E4M3, N, K), b_scale=T(F32, -(-N // 128), kb), out=T(dts[dt], M, N))
    if op == "quantize":
        rows, M, K, dt = a
        return block_quantize(x=T(dts[dt], M, K), codes=T(E4M3, M, K), scales=T(F32, -(-M // rows), -(-K // 128)), rows=rows)
    if op == "rotate":
        dt, rows, D, R, weights = a
        t = {x + "_weight": T(dts[dt], D) for x in weights}
        return paged_norm_rotate(q=T(dts[dt], rows, 32, D), k=T(dts[dt], rows, 8, D), q_out=T(dts[dt], rows, 32, D), k_out=T(dts[dt], rows, 8, D),
                                 cos=T(F32, 99, R // 2), sin=T(F32, 99, R // 2), lengths=T(I32, 9), starts=T(I32, 10), **t)
    dt, code, H, D, page, G, rows = a
    return paged_prefix_attention(q=T(dts[dt], rows, H * G, D), out=T(dts[dt], rows, H * G, D), prefix_table=T(I32, 2, 9), prefix_lengths=T(I32, 2),
                                  members=T(I32, 3), page_table=T(I32, 40, 9), lengths=T(I32, 40), starts=T(I32, 41), **cache(dts[code], 100, H, page, D))


def look(case):
    """The case's launches, the kernels of the code object that they built, and what is wrong with them."""
    import code_objects
    import hip_stub

    with tempfile.TemporaryDirectory() as d:
        os.environ["PTO_WSP_CODEGEN_CACHE_DIR"] = d
        with hip_stub.program(workload_of(case)) as once:
            launches = [(x.entry, x.blocks, x.threads) for x in once()]
        found, wrong = [], []
        for name in os.listdir(os.path.join(d, "hip")):
            path = os.path.join(d, "hip", name)
            for kernel, code in code_objects.kernels(path).items():
                found.append(kernel)
                wrong += [f"{kernel}: {x}" for x in code_objects.ahead_of_restore(code)]
                wrong += [f"{kernel}: {t}" for _, t, _ in code if "Invalid" in t or re.match(r"v_mfma_scale.*, s\d+", t)]
            wrong += [f"{kernel}: {n} bytes of scratch" for kernel, n in code_objects.scratch_bytes(path).items() if n]
    return {"launches": launches, "found": sorted(found), "wrong": wrong}


COMPILERS = ("torch", "system")  # torch's, and ROCm's own
SHARES = 4


@pytest.fixture(scope="module")
def seen():
    """What fresh processes find, by compiler and case."""
    import hip_stub

    hip_stub._library()  # built once, ahead of the processes
    here = os.path.dirname(os.path.abspath(__file__))
    runs = {}
    for compiler in COMPILERS:
        env = dict(os.environ)
        env.pop("PTO_WSP_TEST_WITHOUT_TORCH", None)
        if compiler == "system":
            env["PTO_WSP_TEST_WITHOUT_TORCH"] = "1"
        for share in range(SHARES):
            runs[compiler, share] = subprocess.Popen([sys.executable, __file__, str(share)], env=env, cwd=here, stdout=subprocess.PIPE, stderr=subprocess.PIPE, text=True)
    found = {}
    for (compiler, share), run in runs.items():
        out, err = run.communicate()
        assert run.returncode == 0, err[-3000:]
        for line in out.splitlines():
            if line.startswith("{"):
                r = json.loads(line)
                found[compiler, r["case"]] = r
    return found


@pytest.mark.parametrize("i", range(len(CASES)), ids=["-".join(str(x) for x in c) for c in CASES])
@pytest.mark.parametrize("compiler", COMPILERS)
def test_kernels(seen, compiler, i):
    r = seen[compiler, i]
    assert r["launches"] and {entry for entry, _, _ in r["launches"]} <= set(r["found"])
    if CASES[i][0] == "matmul":
        bm, bn, threads, M, N = CASES[i][1:6]
        assert r["launches"] == [["ptowsp_block_matmul", -(-M // bm) * -(-N // bn), threads]]
    assert not r["wrong"], "; ".join(r["wrong"])


if __name__ == "__main__":
    import conftest  # noqa: F401  (paths, and the absence of torch where that is asked for)

    if not os.environ.get("PTO_WSP_TEST_WITHOUT_TORCH"):
        import torch  # noqa: F401
    for i in range(int(sys.argv[1]), len(CASES), SHARES):
        print(json.dumps({"case": i, **look(CASES[i])}), flush=True)
