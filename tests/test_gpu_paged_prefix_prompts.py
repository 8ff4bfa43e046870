"""GPU tests of paged_prefix_attention where requests have prompts of their own behind the prefixes: units of own tokens
from a list (more than 8192 query rows in the call, of which a request has more than 64 a key head), whole, in several
pieces, and done over.  Tolerances are those of test_gpu_paged_prefix."""

import numpy as np
import pytest

from pto_wsp import ExecutionError, sequential
from test_gpu_paged_prefix import call, case, check, reference, tensors

pytestmark = pytest.mark.gpu


def test_prompts_out_of_range_behind_another_call(gpu):
    """A bad request leaves its rows' entries as an earlier call of the program left that memory: here one whose prefix
    was cut into pieces.  It raises, rows of no request stay, and the same operands put right give right results."""
    rng = np.random.default_rng(1)
    many = case(rng, "bf16", "e4m3", 8, 4, 64, 16, [6000], [0, 70], [20] * 70, [4] * 70, poison=False)
    c = case(rng, "bf16", "e4m3", 2, 16, 64, 16, [100, 40], [0, 2, 3], [300, 90, 150], [200, 40, 100], poison=False)
    t, u = tensors(gpu, many), tensors(gpu, c)
    good = u["lengths"].clone()
    u["lengths"][1] = -1
    prog = sequential(call(t), call(u)).compile(target="hip_gfx950")
    for _ in range(2):
        prog.execute()
        with pytest.raises(ExecutionError, match="paged_prefix_attention"):
            prog.synchronize()
    assert (u["out"][int(c["starts"][-1]):] == 7).all()
    u["lengths"].copy_(good)
    prog.execute()
    prog.synchronize()
    check(many, t, reference(many, 1 / 8))
    check(c, u, reference(c, 1 / 8))
