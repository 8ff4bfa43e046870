"""GPU tests of paged_prefix_attention against a plain form in 64 bits: softmax over a row's prefix and its own tokens.

The tolerance is that of paged_attention's tests (test_gpu_paged) over all the tokens that a row sees, which holds
for each part; joining them multiplies each result with a weight that is off by the scores' error again (an exponent
of the two maxima's difference) and by 6 roundings of 2^-24.  Groups of more than 64 rows a key head run in the kernel
for prompts, with f16 weights for bf16 queries."""

import numpy as np
import pytest

import paged_ref as R
from pto_wsp import ExecutionError, paged_attention, paged_prefix_attention
from test_gpu_paged import HALF, PARTS, PROMPT, T, _dt, _torch, codes_on, go, ints

pytestmark = pytest.mark.gpu


def case(rng, dt, kind, H, G, D, page, prefix, members, lengths, counts, behind=3, poison=True, spread=0.5):
    """Inputs as numpy arrays; what no row may see is filled with NaN codes and scales, or large ones."""
    torch = _torch()
    prefix, members, lengths, counts = (np.asarray(x, int) for x in (prefix, members, lengths, counts))
    held = np.concatenate([prefix, lengths])
    need = -(-held // page)
    pages = int(need.sum()) + 3
    order = rng.permutation(pages)
    width = max(1, int(need.max(initial=0)) + 1)
    table = np.full((len(held), width), 10 ** 6 if poison else 0, np.int64)  # never looked up
    codes, scale = {}, {}
    for x in "kv":
        codes[x] = R.encode(rng.standard_normal((pages, H, page, D)) * 40, kind)
        scale[x] = (0.03 * np.exp(spread * rng.standard_normal((pages, H)))).astype(np.float32)
    live, at = np.zeros((pages, page), bool), 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        live[order[at:at + n]] = (np.arange(n * page) < held[b]).reshape(n, page)
        at += n
    if poison:
        for x in "kv":
            codes[x] = np.where(live[:, None, :, None], codes[x], 0x7F).astype(codes[x].dtype)
            scale[x] = np.where(live.any(1)[:, None], scale[x], np.nan).astype(np.float32)
    starts = np.concatenate([[0], np.cumsum(counts)])
    q = torch.from_numpy(rng.standard_normal((int(starts[-1]) + behind, H * G, D)).astype(np.float32)).to(_dt(dt))
    return {"q": q, "codes": codes, "scale": scale, "prefix_table": table[:len(prefix)], "table": table[len(prefix):], "prefix": prefix,
            "members": members, "lengths": lengths, "starts": starts, "kind": kind, "dt": dt}


def tensors(gpu, c):
    torch = _torch()
    t = {"q": c["q"].to(gpu), "page_table": ints(gpu, c["table"]), "lengths": ints(gpu, c["lengths"]), "starts": ints(gpu, c["starts"]),
         "prefix_table": ints(gpu, c["prefix_table"]), "prefix_lengths": ints(gpu, c["prefix"]), "members": ints(gpu, c["members"])}
    for x in "kv":
        t[x + "_cache"], t[x + "_scale"] = codes_on(gpu, c["codes"][x], c["kind"]), torch.from_numpy(c["scale"][x]).to(gpu)
    t["out"] = torch.full_like(t["q"], 7.0)
    t["lse"] = torch.full(t["q"].shape[:2], 7.0, device=gpu)
    return t


def reference(c, scale):
    """out, lse, and what bounds an evaluation's error, as paged_ref.attend; tokens that the longest row sees."""
    k, v = (R.decode(c["codes"][x], c["kind"]) * c["scale"][x].astype(np.float64)[:, :, None, None] for x in "kv")
    H, D = k.shape[1], k.shape[3]
    q = c["q"].double().numpy()
    rows, HQ, _ = q.shape
    G, longest = HQ // H, 1
    out, lse = np.zeros((rows, HQ, D)), np.full((rows, HQ), -np.inf)
    spread, swing, bulk = np.zeros((rows, HQ, D)), np.zeros((rows, HQ)), np.zeros((rows, HQ, D))

    def held(x, pages, n):
        page = x.shape[2]
        return x[pages[:-(-n // page)]].transpose(1, 0, 2, 3).reshape(H, -1, D)[:, :n]

    ahead = {}
    for g, n in enumerate(c["prefix"]):
        for b in range(c["members"][g], c["members"][g + 1]):
            ahead[b] = (held(k, c["prefix_table"][g], n), held(v, c["prefix_table"][g], n))
    for b, L in enumerate(c["lengths"]):
        kk, vv = held(k, c["table"][b], L), held(v, c["table"][b], L)
        P = 0
        if b in ahead:
            P = ahead[b][0].shape[1]
            kk, vv = np.concatenate([ahead[b][0], kk], 1), np.concatenate([ahead[b][1], vv], 1)
        n = c["starts"][b + 1] - c["starts"][b]
        for i in range(n):
            end, r = P + max(0, L - n + i + 1), c["starts"][b] + i
            longest = max(longest, end)
            if end == 0:
                continue
            kt, vt = kk[:, :end], vv[:, :end]
            x = q[r].reshape(H, G, D)
            with np.errstate(invalid="ignore"):
                s = (x @ kt.transpose(0, 2, 1)) * scale
                m = s.max(-1, keepdims=True)
                e = np.exp(s - m)
                total = e.sum(-1, keepdims=True)
                out[r] = ((e @ vt) / total).reshape(HQ, D)
                lse[r] = (m + np.log(total)).reshape(HQ)
                spread[r] = ((e @ np.abs(vt)) / total).reshape(HQ, D)
                bulk[r] = np.repeat(np.abs(vt).sum(1), G, 0)
                swing[r] = (np.abs(x) @ np.abs(kt).transpose(0, 2, 1)).max(-1).reshape(HQ) * abs(scale)
    return out, lse, spread, swing, bulk, longest


def check(c, t, ref, lse=True):
    out, want, spread, swing, bulk, longest = ref
    dt, D, n = c["dt"], out.shape[-1], int(c["starts"][-1])
    G = c["q"].shape[1] // c["codes"]["k"].shape[1]
    many = max([int(c["starts"][c["members"][g + 1]] - c["starts"][c["members"][g]]) for g in range(len(c["prefix"]))] + [int(np.diff(c["starts"]).max())])
    parts = (PROMPT if many * G > 64 else PARTS)[dt]
    ds = (D + 8) * 2.0 ** -24 * np.maximum(swing, 1.0)
    sums = (longest / 128 + 64 + D + 12) * 2.0 ** -24
    tol = HALF[dt] * np.abs(out) + spread * (4 * ds[..., None] + parts + sums) + bulk * 2.0 ** -30
    tol = tol * (1 + 2 * HALF[dt]) + (2.0 ** -25 if dt == "f16" else 2.0 ** -140)
    got = t["out"].double().cpu().numpy()
    assert np.array_equal(np.isnan(got[:n]), np.isnan(out[:n]))
    off = np.abs(got[:n] - out[:n])
    assert (np.isnan(out[:n]) | (off <= tol[:n])).all(), f"off by {np.nanmax(off / tol[:n]):.3g} of the tolerance"
    assert (got[n:] == 7.0).all()
    if lse:
        a = t["lse"].double().cpu().numpy()
        assert np.array_equal(np.isinf(a[:n]), np.isinf(want[:n])) and (a[n:] == 7.0).all()
        fine = np.isfinite(want[:n])
        ltol = 4 * ds[:n] + sums + 2.0 ** -23 * np.abs(np.where(np.isfinite(want[:n]), want[:n], 0.0))
        assert (np.abs(a[:n] - want[:n])[fine] <= ltol[fine]).all()


def call(t, lse=True, **other):
    return paged_prefix_attention(**{k: T(x) for k, x in t.items() if lse or k != "lse"}, **other)


def attend(gpu, c, scale=None, lse=True):
    t = tensors(gpu, c)
    prog = go(call(t, lse, scale=scale))
    check(c, t, reference(c, scale if scale is not None else 1.0 / np.sqrt(c["q"].shape[-1])), lse)
    return prog, t


SHAPES = [
    # H, G, D, page, prefix lengths, members, lengths, counts
    (1, 1, 64, 16, [1], [0, 1], [1], [1]),
    (2, 4, 128, 16, [33], [0, 4], [1, 31, 33, 5], [1, 1, 1, 1]),
    (2, 7, 80, 8, [260, 17], [0, 2, 5], [5, 260, 17, 1, 2], [1, 1, 1, 1, 1]),
    (1, 16, 256, 64, [300], [0, 3], [64, 1, 9], [1, 1, 1]),
    (1, 40, 64, 32, [130], [0, 2], [130, 3], [1, 3]),
    (3, 2, 16, 1, [40], [0, 2], [9, 1], [1, 1]),
    (2, 5, 96, 24, [100, 0, 47], [0, 1, 2, 4], [3, 30, 25, 1], [1, 1, 1, 1]),
    # requests ahead of the groups and behind them, a group without requests, one without a prefix
    (2, 2, 64, 16, [50, 9, 0, 70], [1, 3, 3, 4, 6], [9, 20, 3, 64, 2, 80, 7], [2, 5, 0, 64, 1, 3, 7]),
    # prompts behind prefixes, idle requests, requests without tokens of their own
    (2, 4, 128, 16, [500], [0, 5], [90, 200, 0, 64, 1], [9, 70, 0, 64, 1]),
    (1, 8, 64, 16, [129, 1000], [0, 2, 3], [150, 40, 50], [150, 0, 33]),
    (2, 3, 48, 128, [200], [0, 2], [200, 129], [130, 129]),
    (1, 24, 128, 16, [70], [0, 2], [70, 20], [40, 3]),
    # more rows than own tokens: the first ones see the prefix alone, or nothing
    (2, 4, 64, 16, [30], [0, 1], [3, 2], [8, 5]),
    # many single tokens behind one long prefix, cut into pieces
    (2, 4, 128, 16, [3000], [0, 40], [5] * 40, [1] * 40),
]


@pytest.mark.parametrize("dt,kind", [("bf16", "e4m3"), ("f16", "i8"), ("f32", "e4m3"), ("bf16", "i8"), ("f32", "i8"), ("f16", "e4m3")])
@pytest.mark.parametrize("shape", range(len(SHAPES)))
def test_prefix(gpu, shape, dt, kind):
    attend(gpu, case(np.random.default_rng(shape), dt, kind, *SHAPES[shape]), lse=shape % 2 == 0)


@pytest.mark.parametrize("dt", ["bf16", "f16", "f32"])
def test_prefix_without_groups(gpu, dt):
    """No group at all, or none of the requests in one: as paged_attention."""
    rng = np.random.default_rng(1)
    attend(gpu, case(rng, dt, "e4m3", 2, 4, 64, 16, [20], [1, 1], [9, 40], [1, 3]))
    c = case(rng, dt, "e4m3", 2, 4, 64, 16, [20], [0, 2], [9, 40], [1, 3])
    t = tensors(gpu, c)
    t |= {"prefix_table": t["prefix_table"][:0], "prefix_lengths": t["prefix_lengths"][:0], "members": t["members"][:1]}
    go(call(t))
    c |= {"prefix": np.zeros(0, int), "members": np.zeros(1, int)}
    check(c, t, reference(c, 1 / 8))


def test_prefix_of_one_is_paged_attention(gpu):
    """A prefix of whole pages: the same requests with the prefix's pages ahead in their own tables."""
    torch = _torch()
    c = case(np.random.default_rng(2), "f32", "i8", 2, 4, 64, 16, [48], [0, 3], [9, 40, 3], [1, 3, 3], poison=False)
    _, t = attend(gpu, c)
    joined = {k: t[k] for k in ("q", "k_cache", "v_cache", "k_scale", "v_scale", "starts")}
    joined["page_table"] = torch.cat([t["prefix_table"][:, :3].expand(3, 3), t["page_table"]], 1).contiguous()
    joined |= {"lengths": t["lengths"] + 48, "out": torch.zeros_like(t["q"]), "lse": torch.zeros_like(t["lse"])}
    go(paged_attention(**{k: T(x) for k, x in joined.items()}))
    n = int(c["starts"][-1])
    assert (joined["out"][:n] - t["out"][:n]).abs().max() < 1e-5 and (joined["lse"][:n] - t["lse"][:n]).abs().max() < 1e-5


@pytest.mark.parametrize("dt", ["bf16", "f16"])
@pytest.mark.parametrize("page", [16, 8])
def test_prefix_scales_far_apart(gpu, page, dt):
    """Pages whose scales differ by more than f16 holds, single tokens and prompts behind them."""
    attend(gpu, case(np.random.default_rng(3), dt, "i8", 2, 4, 64, page, [700, 300], [0, 30, 32], [40] * 30 + [90, 90], [1] * 30 + [60, 3], spread=4.0))


@pytest.mark.parametrize("scale", [-0.2, 0.0, 3.0])
def test_prefix_scale(gpu, scale):
    attend(gpu, case(np.random.default_rng(4), "f32", "e4m3", 1, 4, 64, 16, [90], [0, 2], [9, 40], [1, 30]), scale=scale)


def test_prefix_nan_reaches_the_rows_that_see_it(gpu):
    """A NaN among a prefix's values makes its group's rows NaN in that dim, no other ones."""
    c = case(np.random.default_rng(5), "bf16", "e4m3", 2, 2, 64, 16, [70, 70], [0, 20, 40], [4] * 41, [1] * 40 + [4], poison=False)
    c["codes"]["v"][c["prefix_table"][1, 2], 1, 5, 3] = 0x7F
    _, t = attend(gpu, c)
    got = t["out"].float().cpu().numpy()
    assert np.isnan(got[20:40, 2:, 3]).all() and not np.isnan(got[:20]).any() and not np.isnan(got[40:44]).any()


def test_prefix_shared_by_many(gpu):
    """More query rows than a kernel's list of units has for itself; several groups of prompts."""
    rng = np.random.default_rng(6)
    counts = [1] * 90 + [130, 1, 70, 0, 200]
    attend(gpu, case(rng, "bf16", "e4m3", 2, 8, 128, 16, [900, 17, 2500], [0, 60, 92, 95], [c + 3 for c in counts], counts), lse=False)


@pytest.mark.parametrize("many", [2, 40, 69])
@pytest.mark.parametrize("groups", [1, 2])
def test_prefix_pieces_by_units(gpu, many, groups):
    """Units of a group's rows few (pieces for one workgroup a compute unit), more (for two) and many (beyond that)."""
    members = [0, many // 2, many] if groups == 2 else [0, many]
    attend(gpu, case(np.random.default_rng(11), "bf16", "e4m3", 8, 4, 64, 16, [1500, 777][:groups], members, [20] * many, [16] * many))


def test_prefix_layouts(gpu):
    """Strided queries, results, tables and counts."""
    torch = _torch()
    c = case(np.random.default_rng(7), "bf16", "i8", 2, 4, 80, 16, [100, 30], [0, 2, 3], [20, 5, 40], [3, 1, 40])
    t = tensors(gpu, c)
    rows, HQ, D = t["q"].shape
    t["q"] = torch.zeros((rows, HQ + 1, D + 1), dtype=t["q"].dtype, device=gpu)[:, 1:, 1:].copy_(t["q"])
    t["out"] = torch.full((HQ, rows, 2 * D), 7.0, dtype=t["q"].dtype, device=gpu)[:, :, :D].permute(1, 0, 2)
    t["lse"] = torch.full((HQ, rows), 7.0, device=gpu).t()
    for k in ("starts", "members", "lengths", "prefix_lengths"):
        t[k] = torch.full((len(t[k]), 3), -1, dtype=torch.int32, device=gpu)[:, 1].copy_(t[k])
    for k in ("page_table", "prefix_table"):
        t[k] = torch.full((t[k].shape[0], t[k].shape[1] + 3), -1, dtype=torch.int32, device=gpu)[:, 1:-2].copy_(t[k])
    go(call(t))
    check(c, t, reference(c, 1.0 / np.sqrt(80)))


@pytest.mark.parametrize("what", ["page", "length", "own length", "members", "members beyond", "starts"])
@pytest.mark.parametrize("rows", [1, 70])
def test_prefix_out_of_range(gpu, what, rows):
    c = case(np.random.default_rng(8), "bf16", "e4m3", 2, 2, 64, 16, [70, 50], [0, 2, 3], [90] * 3, [rows] * 3, poison=False)
    t = tensors(gpu, c)
    if what == "page":
        t["prefix_table"][1, 2] = 10 ** 6
    elif what == "length":
        t["prefix_lengths"][0] = 16 * t["prefix_table"].shape[1] + 1
    elif what == "own length":
        t["lengths"][1] = -1
    elif what == "members":
        t["members"] = ints(gpu, [2, 1, 3])
    elif what == "members beyond":
        t["members"] = ints(gpu, [0, 2, 4])
    else:
        t["starts"][3] = len(c["q"]) + 1
    p = call(t).compile(target="hip_gfx950")
    p.execute()
    with pytest.raises(ExecutionError, match="paged_prefix_attention"):
        p.synchronize()


@pytest.mark.parametrize("dt,counts", [("bf16", [1] * 30), ("f16", [1] * 3 + [100, 20]), ("f32", [1, 1, 2])])
def test_prefix_captured(gpu, dt, counts):
    """Captured twice and replayed beside eager runs: every graph keeps a workspace of its own."""
    torch = _torch()
    n = len(counts)
    c = case(np.random.default_rng(9), dt, "e4m3", 2, 4, 64, 16, [800, 90], [0, n - 1, n], [x + 5 for x in counts], counts)
    t = tensors(gpu, c)
    ref = reference(c, 1 / 8)
    prog = call(t).compile(target="hip_gfx950")
    graphs = []
    for _ in range(2):
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            prog.execute()
            prog.synchronize()
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            prog.execute()
        prog.synchronize()
        graphs.append(g)
    eager = None
    for _ in range(3):
        for g in graphs + [None]:
            t["out"].fill_(7.0)
            t["lse"].fill_(7.0)
            torch.cuda.synchronize()
            if g is None:
                prog.execute()
                prog.synchronize()
            else:
                g.replay()
                torch.cuda.synchronize()
            check(c, t, ref)
            eager = t["out"].clone() if eager is None else eager
            assert torch.equal(eager, t["out"])
