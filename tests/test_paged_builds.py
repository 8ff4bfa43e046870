"""The kernels that a build without a GPU makes of a paged operator are those that a run of it launches."""

import re

import pytest

import hip_stub
from pto_wsp import DType, sequential
from pto_wsp._hip import NativeProgram
from pto_wsp.ir_bridge import workload_to_codegen_ir
from test_paged_host import attend, cache, plan, store


def sources(workload, steps=1):
    prog = NativeProgram(workload_to_codegen_ir(workload, "build").module)
    return [prog.precompile(i) for i in range(steps)]


# Tiles of 16 rows of the kernel for few rows, and of the one for prompts (32 only in 16 bits, up to head size 128, over
# pages of a multiple of 16; beside prompts few rows are single tokens, of up to 16 heads in one tile of 16).
@pytest.mark.parametrize("dt,rows,batch,G,D,page,few,prompts", [
    (DType.BF16, 2048, 4, 4, 128, 16, 1, 2), (DType.BF16, 2048, 4, 20, 128, 16, 2, 2), (DType.F16, 700, 2, 6, 96, 16, 1, 2),
    (DType.F32, 2048, 4, 4, 48, 8, 1, 1), (DType.BF16, 2048, 4, 4, 128, 24, 1, 1),
    (DType.BF16, 300, 4, 2, 112, 32, 2, None), (DType.BF16, 9, 4, 3, 128, 40, 1, None), (DType.F32, 300, 4, 2, 112, 32, 1, None),
])
def test_attention(dt, rows, batch, G, D, page, few, prompts):
    def call():
        return attend(rows=rows, batch=batch, G=G, D=D, dt=dt, c=cache(page=page, D=D))

    (source,) = sources(call())
    kinds = set(re.findall(rf"Attend<{D}, {page}, {G}, (\d), \d, 0, false, false, true, (true|false)>", source))
    assert kinds == {(str(few), "false")} | ({(str(prompts), "true")} if prompts else set())
    with hip_stub.program(call()) as once:
        entries = [x.entry for x in once()]
    assert sorted(re.findall(r"void (ptowsp_\w+)\(", source)) == sorted(entries)


def test_numbers():
    """One source a step, in order."""
    found = sources(sequential(plan(), store(), attend()), 3)
    for name, source in zip(("ptowsp_paged_plan(", "ptowsp_paged_store(", "ptowsp_paged_attention("), found):
        assert name in source
