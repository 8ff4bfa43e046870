"""Kernels of paged_attention as a run builds them (on the CPU: launches are recorded instead of run),
where the registers are fewest: head sizes that end inside 64 dims, pages that end inside 16 tokens,
groups that leave rows of a wave empty.

Where only some lanes take a branch, the compiler may put a copy or a spill of a register at the branch's end
before the other lanes go on.  Those lanes then read what the register's new place held before."""

import glob
import os
import subprocess
import sys

import pytest

import code_objects
import hip_stub
from test_paged_host import T, attend, cache
from pto_wsp import DType

DT = {"bf16": DType.BF16, "f16": DType.F16, "f32": DType.F32, "e4m3": DType.F8E4M3, "i8": DType.I8}


def _text(bad):
    return "; ".join(f"{name}: {what}" for name, what in bad)


def _check(tmp_path, monkeypatch, dt, code, D, page, G, window, lse, prompts):
    monkeypatch.setenv("PTO_WSP_CODEGEN_CACHE_DIR", str(tmp_path))
    rows, heads = (9000, 3) if prompts else (4, 3)
    other = {"lse": T(DType.F32, rows, heads * G)} if lse else {}
    with hip_stub.program(attend(rows=rows, heads=heads, G=G, D=D, batch=4, dt=DT[dt], c=cache(DT[code], 100, heads, page, D), window=window, **other)) as once:
        entries = [x.entry for x in once()]
    assert ("ptowsp_paged_attention_prompts" in entries) == prompts
    objects = glob.glob(str(tmp_path / "hip" / "*.hsaco"))
    assert objects, "the kernels were built before this test"
    for path in objects:
        code = code_objects.kernels(path)
        assert set(entries) <= set(code)
        bad = [(name, x) for name, instructions in code.items() for x in code_objects.ahead_of_restore(instructions)]
        assert not bad, _text(bad)
        spilled = {name: n for name, n in code_objects.scratch_bytes(path).items() if n}
        assert not spilled, spilled


# Built without the two rules that keep this so, each of these had copies or spills in such places.
@pytest.mark.parametrize("dt,code,D,page,G,window,lse,prompts", [
    ("bf16", "i8", 240, 8, 7, 9, False, False), ("f16", "i8", 240, 8, 40, 9, False, False), ("bf16", "i8", 176, 8, 16, 9, False, False),
    ("f32", "e4m3", 176, 24, 24, 0, False, False), ("f16", "e4m3", 112, 24, 40, 0, True, False), ("f32", "i8", 144, 64, 5, 9, True, False),
    ("f16", "e4m3", 96, 24, 24, 0, False, False), ("bf16", "i8", 112, 64, 24, 0, True, False), ("f32", "i8", 96, 8, 16, 0, True, False),
    ("bf16", "i8", 208, 1, 12, 0, True, True), ("f32", "e4m3", 208, 8, 12, 0, True, True), ("f16", "i8", 144, 8, 2, 0, False, True),
    ("bf16", "i8", 96, 24, 40, 9, False, True), ("f32", "i8", 144, 64, 40, 0, False, True), ("bf16", "i8", 128, 8, 40, 0, False, True),
])
def test_lanes_keep_their_registers(tmp_path, monkeypatch, dt, code, D, page, G, window, lse, prompts):
    _check(tmp_path, monkeypatch, dt, code, D, page, G, window, lse, prompts)


# Spilled registers, though at safe places.
@pytest.mark.parametrize("dt,code,D,page,G,window,lse,prompts", [
    ("f32", "i8", 128, 8, 2, 0, False, False), ("f32", "e4m3", 256, 8, 7, 0, True, False), ("f32", "i8", 256, 16, 4, 9, True, True),
    ("bf16", "e4m3", 128, 16, 24, 9, False, False), ("f16", "e4m3", 96, 16, 24, 9, True, True),
])
def test_no_register_is_spilled(tmp_path, monkeypatch, dt, code, D, page, G, window, lse, prompts):
    _check(tmp_path, monkeypatch, dt, code, D, page, G, window, lse, prompts)


@pytest.mark.parametrize("code", ["i8", "e4m3"])
@pytest.mark.parametrize("page", [8, 16, 24])
@pytest.mark.parametrize("D", [80, 128, 256])
@pytest.mark.parametrize("window", [9, 0])
def test_float32(tmp_path, monkeypatch, code, D, page, window):
    _check(tmp_path, monkeypatch, "f32", code, D, page, 7, window, D == 80, page == 24 and window > 0)


def test_the_system_compiler(tmp_path):
    """The same of the kernels that hiprtc of ROCm itself makes; torch brings its own."""
    if os.environ.get("PTO_WSP_TEST_WITHOUT_TORCH"):
        pytest.skip("runs without torch already")
    run = subprocess.run([sys.executable, "-m", "pytest", "-q", "-p", "no:cacheprovider", "--basetemp", str(tmp_path / "t"), "-k", "lanes_keep", __file__],
                         env=dict(os.environ, PTO_WSP_TEST_WITHOUT_TORCH="1"), capture_output=True, text=True)
    assert run.returncode == 0 and "15 passed" in run.stdout, run.stdout[-3000:]


def test_the_search_finds_them():
    code = [(0, "s_and_saveexec_b64 s[2:3], vcc", None), (4, "s_cbranch_execz 2", 16), (8, "global_load_dword v1, v[2:3], off", None),
            (16, "s_mov_b32 s5, s6", None), (20, "scratch_store_dword off, v9, off", None), (28, "s_or_b64 exec, exec, s[2:3]", None)]
    assert code_objects.ahead_of_restore(code) == ["scratch_store_dword off, v9, off"]
    assert code_objects.ahead_of_restore(code[:4] + [(20, "s_or_b64 exec, exec, s[2:3]", None), (24, "v_mov_b32_e32 v1, v2", None)]) == []
