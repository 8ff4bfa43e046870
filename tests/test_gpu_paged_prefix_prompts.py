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


def attend(gpu, c, scale=None, lse=True):
    """The call's launches are those with a list of units, and some request's rows are on it."""
    HQ, H = c["q"].shape[1], c["codes"]["k"].shape[1]
    assert c["q"].shape[0] * HQ > 8192 and np.diff(c["starts"]).max() * (HQ // H) > 64
    t = tensors(gpu, c)
    prog = call(t, lse, scale=scale).compile(target="hip_gfx950")
    prog.execute()
    prog.synchronize()
    assert prog.stats.launches == 4  # the list, both parts, cut units, the join
    check(c, t, reference(c, scale if scale is not None else 1.0 / np.sqrt(c["q"].shape[-1])), lse)
    return prog, t


SHAPES = [
    # H, G, D, page, prefix lengths, members, lengths, counts
    # several prompts behind one prefix, single tokens, a request without rows and one without a prefix beside them
    (2, 8, 128, 16, [300], [0, 5], [150, 1, 40, 400, 9, 200], [150, 1, 0, 260, 9, 140]),
    # several groups, one without a prefix, one without requests; requests ahead of the groups and behind them
    (4, 4, 64, 16, [700, 0, 33, 90], [1, 3, 4, 4, 6], [110, 300, 5, 129, 70, 30, 200], [110, 128, 1, 129, 65, 30, 100]),
    # odd pages, of which tiles are not made, and heads that end inside 64 dims
    (2, 8, 80, 24, [100, 50], [0, 2, 3], [200, 70, 300], [200, 30, 290]),
    (1, 20, 64, 1, [65], [0, 2], [230, 250], [200, 220]),
    (2, 6, 256, 8, [129], [0, 3], [400, 17, 333], [390, 17, 300]),
    # one prompt over many tokens: units in several pieces
    (1, 32, 128, 16, [600], [0, 1], [5000], [260]),
    (2, 16, 64, 32, [40, 3000], [0, 1, 3], [4097, 900, 1], [258, 17, 1]),
    # more rows than own tokens: the first ones see the prefix alone, or nothing
    (2, 8, 64, 16, [30], [0, 1], [100, 60], [300, 250]),
    # more query heads of a key head than a wave has rows
    (1, 70, 64, 16, [50], [0, 2], [150, 100], [90, 30]),
]


@pytest.mark.parametrize("shape,dt,kind,lse", [
    (0, "bf16", "e4m3", True), (0, "f32", "i8", False), (1, "f16", "i8", True), (2, "bf16", "i8", False), (3, "f16", "e4m3", False), (4, "f32", "e4m3", True),
    (5, "bf16", "e4m3", False), (6, "f16", "e4m3", True), (6, "f32", "i8", False), (7, "bf16", "i8", True), (8, "bf16", "e4m3", False),
])
def test_prompts(gpu, shape, dt, kind, lse):
    attend(gpu, case(np.random.default_rng(100 + shape), dt, kind, *SHAPES[shape]), lse=lse)


@pytest.mark.parametrize("dt", ["bf16", "f16"])
@pytest.mark.parametrize("lengths,counts", [([400, 300, 1], [260, 200, 1]), ([3000, 7], [264, 7])])
def test_prompts_with_scales_far_apart(gpu, lengths, counts, dt):
    """Pages whose scales differ by more than f16 holds, among own tokens and in the prefix: units are done over, whole
    ones and pieces."""
    attend(gpu, case(np.random.default_rng(7), dt, "i8", 2, 16, 64, 16, [500], [0, len(lengths)], lengths, counts, spread=4.0))


@pytest.mark.parametrize("scale", [-0.2, 0.0])
def test_prompts_scale(gpu, scale):
    attend(gpu, case(np.random.default_rng(8), "bf16", "e4m3", 2, 16, 64, 16, [90], [0, 2], [200, 140], [170, 130]), scale=scale)


def test_prompts_nan_reaches_the_rows_that_see_it(gpu):
    """A NaN among a request's own values: the rows from its position on, of its key head, in its dim."""
    c = case(np.random.default_rng(9), "bf16", "e4m3", 2, 16, 64, 16, [70], [0, 2], [300, 100], [200, 90], poison=False)
    c["codes"]["v"][c["table"][0, 10], 1, 4, 3] = 0x7F  # position 164, row 64
    _, t = attend(gpu, c)
    got = t["out"].float().cpu().numpy()[:290]
    assert np.isnan(got[64:200, 16:, 3]).all() and np.isnan(got).sum() == 136 * 16


def test_prompts_captured(gpu):
    """Captured and replayed beside eager runs, the same to the bit."""
    import torch

    c = case(np.random.default_rng(10), "bf16", "e4m3", 2, 16, 64, 16, [800], [0, 3], [1200, 90, 1], [260, 70, 1])
    t = tensors(gpu, c)
    ref = reference(c, 1 / 8)
    prog = call(t).compile(target="hip_gfx950")
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        prog.execute()
        prog.synchronize()
    check(c, t, ref)
    first = t["out"].clone()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        prog.execute()
    prog.synchronize()
    for _ in range(3):
        for replay in (True, False):
            t["out"].fill_(7.0)
            t["lse"].fill_(7.0)
            torch.cuda.synchronize()
            if replay:
                g.replay()
                torch.cuda.synchronize()
            else:
                prog.execute()
                prog.synchronize()
            check(c, t, ref)
            assert torch.equal(first, t["out"])


def test_more_groups_than_threads(gpu):
    """300 groups with more rows than the kernel for few takes, of one request or two, some without a prefix and some
    without rows: each workgroup finds its piece among them."""
    rng = np.random.default_rng(11)
    counts = rng.integers(17, 24, size=400)
    counts[rng.permutation(400)[:40]] = 0
    counts[7] = 90
    members = np.concatenate([[0], np.cumsum(np.arange(300) % 3 == 0) + np.arange(1, 301)])
    prefix = rng.integers(0, 200, size=300)
    prefix[rng.permutation(300)[:30]] = 0
    attend(gpu, case(rng, "bf16", "e4m3", 1, 4, 64, 16, prefix, members, counts + rng.integers(0, 60, size=400), counts))
