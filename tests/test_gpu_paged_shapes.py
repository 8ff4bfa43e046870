"""GPU tests of paged_attention over head sizes, groups and pages that fill no registers evenly, and of its
prompts, against the plain form in 64 bits (paged_ref).

Each row is held to the error of the kernel that it runs in (test_gpu_paged derives them): weights as two bf16 parts
(three for float32), or, for a prompt in tiles, as one f16 (two for f16 outputs).  A call gives the same bits
every time: no sum is taken in an order that changes."""

import numpy as np
import pytest

import paged_ref as R
import test_gpu_paged as G
from pto_wsp import DType, Tensor, paged_attention, paged_store

pytestmark = pytest.mark.gpu


def tolerance(c, ref):
    """Of each output, and of each lse."""
    out, lse, spread, swing, bulk = ref
    rows, heads, D = out.shape
    group, page = heads // c["codes"]["k"].shape[1], c["codes"]["k"].shape[2]
    counts, few = np.diff(c["starts"]), max(1, 64 // group)
    prompts = c["q"].shape[0] - len(counts) >= few and c["q"].shape[0] * heads > 8192
    tiled = np.repeat(counts > few, counts) & bool(prompts and c["dt"] != "f32" and D <= 128 and page % 16 == 0)
    parts = np.where(tiled, G.PROMPT[c["dt"]], G.PARTS[c["dt"]])[:, None, None]
    n = int(max(c["lengths"].max(initial=0), 1))
    ds = (D + 8) * 2.0 ** -24 * np.maximum(swing, 1.0)
    sums = (n / 128 + 64 + D) * 2.0 ** -24
    tol = G.HALF[c["dt"]] * np.abs(out) + spread * (2 * ds[..., None] + parts + sums) + bulk * np.where(tiled, 2.0 ** -30, 0.0)[:, None, None]
    tol = tol * (1 + 2 * G.HALF[c["dt"]]) + (2.0 ** -25 if c["dt"] == "f16" else 2.0 ** -140)
    return tol, 2 * ds + sums + 2.0 ** -23 * np.abs(np.where(np.isfinite(lse), lse, 0.0))


def check(c, t, ref):
    n = int(c["starts"][-1])
    ref = tuple(x[:n] for x in ref)
    tol, ltol = tolerance(c, ref)
    got, lse = t["out"].double().cpu().numpy(), t["lse"].double().cpu().numpy()
    assert np.array_equal(np.isnan(got[:n]), np.isnan(ref[0]))
    off = np.abs(got[:n] - ref[0])
    bad = ~(np.isnan(ref[0]) | (off <= tol))
    assert not bad.any(), f"off by {np.nanmax(off / tol):.3g} of the tolerance, first at {np.argwhere(bad)[0]}, heads {np.unique(np.argwhere(bad)[:, 1])}"
    assert (got[n:] == 7.0).all() and (lse[n:] == 7.0).all()
    assert np.array_equal(np.isinf(lse[:n]), np.isinf(ref[1]))
    fine = np.isfinite(ref[1])
    assert (np.abs(lse[:n] - ref[1])[fine] <= ltol[fine]).all()


def attend(gpu, monkeypatch, dt, kind, H, group, D, page, lengths, counts, window, many, seed, change=None):
    """A call with lse, three times, and one without."""
    torch = G._torch()
    monkeypatch.setattr(G, "_rows_behind", G._behind["many" if many else "few"])
    c = G._attend_case(np.random.default_rng(seed), dt, kind, H, group, D, page, lengths, counts, poison=not window)
    if change:
        change(c)
    t = G._attend_tensors(gpu, c)
    w = {k: G.T(x) for k, x in t.items()}
    prog = paged_attention(**w, window=window).compile(target="hip_gfx950")
    first, ref = None, G._reference(c, 1.0 / np.sqrt(D), window)
    for _ in range(3):
        t["out"].fill_(7.0), t["lse"].fill_(7.0)
        prog.execute()
        prog.synchronize()
        check(c, t, ref)
        now = t["out"].clone(), t["lse"].clone()
        first = first or now
        assert all(torch.equal(a.nan_to_num(nan=3.0), b.nan_to_num(nan=3.0)) for a, b in zip(first, now))
    t["out"].fill_(7.0)
    G.go(paged_attention(**{k: x for k, x in w.items() if k != "lse"}, window=window))
    check(c, t, ref)
    return prog


FEW = ([700, 60, 311, 200], [3, 1, 2, 2])
MIXED = ([260, 60, 140, 33], [190, 1, 2, 33])


@pytest.mark.parametrize("dt,kind,group,D,page,window,many", [
    ("bf16", "i8", 7, 240, 8, 250, False), ("f16", "i8", 40, 240, 8, 90, False), ("bf16", "e4m3", 4, 176, 16, 0, False),
    ("f32", "e4m3", 24, 176, 24, 0, False), ("f16", "e4m3", 40, 112, 24, 0, False), ("f32", "i8", 5, 144, 64, 90, False),
    ("bf16", "i8", 24, 112, 64, 0, False), ("f32", "i8", 16, 96, 8, 0, False), ("f16", "i8", 3, 208, 1, 0, False),
    ("f32", "i8", 2, 128, 8, 0, False), ("f32", "e4m3", 7, 256, 8, 0, False), ("f32", "i8", 6, 256, 24, 0, False),
    ("f32", "e4m3", 4, 128, 24, 0, False), ("bf16", "e4m3", 24, 128, 16, 90, False),
    ("bf16", "i8", 12, 208, 1, 0, True), ("f32", "e4m3", 12, 208, 8, 0, True), ("f16", "i8", 2, 144, 8, 0, True),
    ("bf16", "i8", 40, 96, 24, 90, True), ("f32", "i8", 40, 144, 64, 0, True), ("bf16", "e4m3", 5, 240, 16, 90, True),
    ("bf16", "i8", 1, 112, 16, 90, True), ("f16", "e4m3", 24, 96, 16, 90, True), ("f32", "i8", 4, 256, 16, 90, True),
    ("f16", "i8", 7, 80, 32, 0, True), ("bf16", "e4m3", 3, 48, 16, 40, True),
])
def test_head_sizes(gpu, monkeypatch, dt, kind, group, D, page, window, many):
    """Single tokens and a few, and (many) prompts beside them."""
    attend(gpu, monkeypatch, dt, kind, 2, group, D, page, *(MIXED if many else FEW), window, many, D + group)


@pytest.mark.parametrize("kind", ["i8", "e4m3"])
@pytest.mark.parametrize("group,D,page,window,many", [
    (7, 80, 8, 250, False), (7, 80, 8, 250, True), (4, 128, 24, 33, False), (5, 256, 8, 500, False), (5, 256, 8, 33, True), (3, 96, 24, 250, True),
    (1, 16, 40, 250, False), (24, 64, 1, 100, False),
])
def test_float32_windows_over_odd_pages(gpu, monkeypatch, kind, group, D, page, window, many):
    attend(gpu, monkeypatch, "f32", kind, 2, group, D, page, *(MIXED if many else FEW), window, many, D + group)


def test_float32_window_of_single_tokens(gpu, monkeypatch):
    """7 heads of 80 over 8-token pages, 37 requests of one to three tokens."""
    rng = np.random.default_rng(11)
    counts = rng.integers(1, 4, 37)
    attend(gpu, monkeypatch, "f32", "i8", 2, 7, 80, 8, np.maximum(counts, rng.integers(1, 5001, 37)), counts, 1500, False, 12)


@pytest.mark.parametrize("page", [64, 40])
@pytest.mark.parametrize("dt,many", [("bf16", False), ("bf16", True), ("f32", True)])
def test_tokens_far_apart(gpu, monkeypatch, dt, many, page):
    """Pages whose last tokens lie beyond 2^31 bytes from their first ones: two pages of one head, keys and values
    between each other's rows."""
    torch = G._torch()
    monkeypatch.setattr(G, "_rows_behind", G._behind["many" if many else "few"])
    D, step = 64, (1 << 31) // (page - 3) // 16 * 16
    c = G._attend_case(np.random.default_rng(page), dt, "e4m3", 1, 4, D, page, [2 * page - 3], [70 if many else 2], poison=False)
    t = G._attend_tensors(gpu, c)
    assert t["k_cache"].shape[0] == 5 and (page - 1) * step >= 1 << 31 and step <= 1 << 26
    pool = torch.zeros(page * step, dtype=torch.int8, device=gpu)
    for i, x in enumerate(("k_cache", "v_cache")):
        far = torch.as_strided(pool, (5, 1, page, D), (2 * D, 2 * D, step, 1), i * D)
        t[x] = far.copy_(t[x].view(torch.int8)).view(t[x].dtype)
    G.go(paged_attention(**{k: G.T(x) for k, x in t.items()}))
    check(c, t, G._reference(c, 0.125, 0))


def test_operands_that_share_memory(gpu):
    """Parts of one torch tensor, and host arrays that are copied back whole."""
    torch = G._torch()
    c = G._attend_case(np.random.default_rng(1), "bf16", "e4m3", 2, 2, 64, 16, [60], [4])
    t = G._attend_tensors(gpu, c)
    rows = t["q"].shape[0]
    both = torch.zeros((rows + 1, 4, 64), dtype=torch.bfloat16, device=gpu)
    t["q"] = both[1:].copy_(t["q"])
    with pytest.raises(RuntimeError, match="out is written and lies where q does"):
        paged_attention(**{k: G.T(x) for k, x in dict(t, out=both[:-1]).items()}).compile(target="hip_gfx950").execute()
    wide = torch.full((rows, 8, 64), 7.0, dtype=torch.bfloat16, device=gpu)
    t["q"], t["out"] = wide[:, :4].copy_(t["q"]), wide[:, 4:]
    G.go(paged_attention(**{k: G.T(x) for k, x in t.items()}))
    check(c, t, G._reference(c, 0.125, 0))

    pool, x = np.zeros((3, 2, 2, 16, 64), np.int8), np.zeros((5, 2, 64), np.float32)
    host = {"k": x, "v": x, "slots": np.arange(5, dtype=np.int32), "k_cache": pool[:, 0], "v_cache": pool[:, 1],
            "k_scale": np.ones((3, 2), np.float32), "v_scale": np.ones((3, 2), np.float32)}
    kinds = {np.dtype(np.float32): DType.F32, np.dtype(np.int32): DType.I32, np.dtype(np.int8): DType.I8}
    w = paged_store(**{k: Tensor(data=a, shape=a.shape, dtype=kinds[a.dtype]) for k, a in host.items()})
    with pytest.raises(RuntimeError, match="k_cache and v_cache are written and share host memory"):
        w.compile(target="hip_gfx950").execute()


# Windows shorter than a tile of 64 tokens, equal to it, beyond it and beyond every context; units of 4 * (32 / group) rows.
@pytest.mark.parametrize("dt,kind,group,D,page,window", [
    ("f16", "i8", 4, 128, 16, 100), ("f16", "e4m3", 5, 64, 32, 64), ("bf16", "i8", 5, 128, 64, 1), ("bf16", "e4m3", 4, 128, 16, 64),
    ("bf16", "i8", 1, 64, 16, 33), ("f16", "i8", 12, 96, 48, 5000), ("bf16", "e4m3", 40, 64, 16, 200),
])
def test_windows_of_prompts(gpu, monkeypatch, dt, kind, group, D, page, window):
    attend(gpu, monkeypatch, dt, kind, 2, group, D, page, [260, 60, 140, 400], [190, 1, 140, 77], window, True, window)


@pytest.mark.parametrize("dt,kind,window", [("bf16", "e4m3", 3000), ("f16", "i8", 4500), ("bf16", "i8", 0)])
def test_prompts_in_pieces(gpu, monkeypatch, dt, kind, window):
    """Contexts so long that a unit is cut, whose pieces the last launch joins."""
    attend(gpu, monkeypatch, dt, kind, 1, 4, 128, 16, [9000, 40], [130, 17], window, True, 5)


@pytest.mark.parametrize("dt", ["bf16", "f16"])
@pytest.mark.parametrize("window,context", [(25, 200), (0, 200), (3000, 6000)])
def test_nan_in_prompts(gpu, monkeypatch, dt, window, context):
    """A NaN among the values and one among the keys: rows whose window holds them, and those alone, have them."""
    def change(c):
        table, page = c["table"][0], c["codes"]["v"].shape[2]
        for token, what in ((context - 60, "v"), (context - 40, "k")):
            at, off = divmod(token, page)
            c["codes"][what][table[at], 1, off, 5] = 0x7F

    attend(gpu, monkeypatch, dt, "e4m3", 2, 4, 64, 16, [context, 30], [100, 1], window, True, context, change)


@pytest.mark.parametrize("dt,kind,D,page", [("bf16", "e4m3", 128, 16), ("f16", "i8", 64, 8), ("f32", "i8", 80, 16)])
def test_several_tokens_in_few_rows(gpu, monkeypatch, dt, kind, D, page):
    """Up to 64 rows a key head: one unit or several, to the accuracy of single tokens."""
    attend(gpu, monkeypatch, dt, kind, 2, 4, D, page, [300, 77, 16, 41], [16, 5, 16, 1], 0, False, D)
