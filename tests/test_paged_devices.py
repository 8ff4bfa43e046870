"""A program of paged operators keeps to the GPU of its first run (on the CPU: launches are recorded)."""

import pytest

import hip_stub
from test_paged_host import I32, T, attend, plan


@pytest.mark.parametrize("make", [lambda: attend(), lambda: plan(5000, 8, 9), lambda: attend(rows=9000, batch=5000, page_table=T(I32, 5000, 4))])
def test_another_gpu(make):
    with hip_stub.program(make()) as once:
        want = [x.entry for x in once()]
        try:
            hip_stub._lib.stub_device(1)
            with pytest.raises(RuntimeError, match="workspace is on GPU 0, the current one is 1"):
                once()
        finally:
            hip_stub._lib.stub_device(0)
        assert [x.entry for x in once()] == want


def test_each_program_its_gpu():
    try:
        hip_stub._library()
        with hip_stub.program(attend()) as once:
            hip_stub._lib.stub_device(3)
            assert once() and once()
    finally:
        hip_stub._lib.stub_device(0)
