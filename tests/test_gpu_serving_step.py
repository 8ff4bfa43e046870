"""A serving step's operators together on the GPU: activations in 8 bits, the projection to queries, keys and values,
pages for the new tokens, norm and rotation where they lie, the store, attention behind shared prefixes, and the
projection back.  Each step's result is checked against its plain form, given what the steps before it left."""

import numpy as np
import pytest

import block_ref as B
import paged_ref as R
import test_gpu_paged_prefix as prefix_tests
from pto_wsp import (block_matmul, block_quantize, paged_norm_rotate, paged_plan, paged_prefix_attention, paged_store, sequential)
from test_gpu_blocks import U, bits, f64
from test_gpu_paged import HALF, T, _dt, _torch, codes_of, codes_on, go, ints, same_codes

pytestmark = pytest.mark.gpu
H, G, D, PAGE, WIDTH = 2, 4, 64, 16, 320


def step_case(gpu, counts, cached, prefix, members, seed, dt="bf16"):
    torch = _torch()
    rng = np.random.default_rng(seed)
    counts, cached, prefix = (np.asarray(x) for x in (counts, cached, prefix))
    rows, total = int(counts.sum()) + 3, cached + counts
    held, need, shared = -(-cached // PAGE), -(-total // PAGE), -(-prefix // PAGE)
    pages = int(need.sum() + shared.sum()) + 2
    order = rng.permutation(pages)
    table, width = np.full((len(counts), int(need.max()) + 1), -1), int(held.sum())
    table[np.arange(table.shape[1])[None] < held[:, None]] = order[:width]
    ptable = np.full((len(prefix), int(shared.max()) + 1), -1)
    ptable[np.arange(ptable.shape[1])[None] < shared[:, None]] = order[width:width + int(shared.sum())]
    free = order[width + int(shared.sum()):]
    t = {"lengths": ints(gpu, cached), "counts": ints(gpu, counts), "page_table": ints(gpu, table), "free_pages": ints(gpu, free), "used": ints(gpu, [0]),
         "new_lengths": ints(gpu, np.zeros(len(counts))), "new_used": ints(gpu, [0]), "starts": ints(gpu, np.zeros(len(counts) + 1)),
         "slots": ints(gpu, np.full(rows, -2)), "prefix_table": ints(gpu, ptable), "prefix_lengths": ints(gpu, prefix), "members": ints(gpu, members)}
    offsets = np.zeros(len(counts), int)
    for g in range(len(prefix)):
        offsets[members[g]:members[g + 1]] = prefix[g]
    t["offsets"] = ints(gpu, offsets)
    for x in "kv":
        t[x + "_cache"] = codes_on(gpu, R.encode(rng.standard_normal((pages, H, PAGE, D)) * 40, "e4m3"), "e4m3")
        t[x + "_scale"] = torch.from_numpy((0.03 * np.exp(0.3 * rng.standard_normal((pages, H)))).astype(np.float32)).to(gpu)
    wide = H * (G + 2) * D
    t["x"] = torch.from_numpy(rng.standard_normal((rows, WIDTH)).astype(np.float32)).to(gpu).to(_dt(dt))

    def codes(n, k, name, blocks):
        t[name] = codes_on(gpu, np.zeros((n, k), np.uint8), "e4m3")
        t[name + "_scale"] = torch.zeros((blocks, B.blocks(k)), device=gpu)

    codes(rows, WIDTH, "x8", rows)
    codes(rows, H * G * D, "y8", rows)
    for name, n, k in (("w_in", wide, WIDTH), ("w_out", WIDTH, H * G * D)):
        codes(n, k, name, B.blocks(n))
        w = torch.from_numpy((rng.standard_normal((n, k)) / np.sqrt(k)).astype(np.float32)).to(gpu)
        go(block_quantize(x=T(w), codes=T(t[name]), scales=T(t[name + "_scale"]), rows=128))
    t["qkv"] = torch.zeros((rows, wide), dtype=_dt(dt), device=gpu)
    t["y"] = torch.zeros((rows, H * G * D), dtype=_dt(dt), device=gpu)
    t["out"] = torch.zeros((rows, WIDTH), dtype=_dt(dt), device=gpu)
    for x in "qk":
        t[x + "_weight"] = torch.from_numpy((1 + 0.2 * rng.standard_normal(D)).astype(np.float32)).to(gpu).to(_dt(dt))
    angles = np.outer(np.arange(int((total + offsets).max()) + 1), 10000.0 ** (-np.arange(D // 2) / (D // 2)))
    t["cos"], t["sin"] = (torch.from_numpy(f(angles).astype(np.float32)).to(gpu) for f in (np.cos, np.sin))
    return t


def parts(t):
    rows = t["x"].shape[0]
    heads = t["qkv"].view(rows, H * (G + 2), D)
    return heads[:, :H * G], heads[:, H * G:H * (G + 1)], heads[:, H * (G + 1):]


def steps(t):
    """The operators of the step, in order."""
    w = {k: T(x) for k, x in t.items()}
    q, k, v = (T(x) for x in parts(t))
    y = T(t["y"].view(-1, H * G, D))
    cache = {n: w[n] for n in ("k_cache", "v_cache", "k_scale", "v_scale")}
    return [block_quantize(x=w["x"], codes=w["x8"], scales=w["x8_scale"]),
            block_matmul(a=w["x8"], a_scale=w["x8_scale"], b=w["w_in"], b_scale=w["w_in_scale"], out=w["qkv"]),
            paged_plan(page_size=PAGE, **{n: w[n] for n in ("lengths", "counts", "page_table", "free_pages", "used", "new_lengths", "new_used", "starts", "slots")}),
            paged_norm_rotate(q=q, k=k, q_out=q, k_out=k, cos=w["cos"], sin=w["sin"], lengths=w["new_lengths"], starts=w["starts"], offsets=w["offsets"],
                              q_weight=w["q_weight"], k_weight=w["k_weight"]),
            paged_store(k=k, v=v, slots=w["slots"], **cache),
            paged_prefix_attention(q=q, out=y, prefix_table=w["prefix_table"], prefix_lengths=w["prefix_lengths"], members=w["members"], page_table=w["page_table"],
                                   lengths=w["new_lengths"], starts=w["starts"], **cache),
            block_quantize(x=w["y"], codes=w["y8"], scales=w["y8_scale"]),
            block_matmul(a=w["y8"], a_scale=w["y8_scale"], b=w["w_out"], b_scale=w["w_out_scale"], out=w["out"])]


def check_product(t, a, b, out, dt):
    args = [bits(t[a]), t[a + "_scale"].cpu().numpy(), bits(t[b]), t[b + "_scale"].cpu().numpy()]
    want, size = B.matmul(*args)
    bound = HALF[dt] * np.abs(want) + size * (2 * 128 + 4 + 2 * args[1].shape[1]) * U + 7 * 2.0 ** -13 * (1 + HALF[dt]) * B.most(*args)
    assert (np.abs(f64(out) - want) <= bound).all()


def check_codes(t, x, name):
    want, scale = B.quantize(f64(t[x]), 1)
    assert np.array_equal(bits(t[name]), want) and np.array_equal(f64(t[name + "_scale"]), scale)


def run_and_check(t, dt="bf16"):
    """One operator at a time, each checked; the tensors as the whole step leaves them."""
    before = {k: x.clone() for k, x in t.items()}
    first, product, plan, rotate, store, attend, second, back = steps(t)
    go(first)
    check_codes(t, "x", "x8")
    go(product)
    check_product(t, "x8", "w_in", t["qkv"], dt)
    go(plan)
    old = {k: before[k].cpu().numpy() for k in ("lengths", "counts", "page_table", "free_pages")}
    want = R.plan(old["lengths"], old["counts"], old["page_table"], old["free_pages"], 0, PAGE, len(t["slots"]))
    for k, x in want.items():
        assert np.array_equal(t[k].cpu().numpy(), x), k
    rows = int(want["starts"][-1])
    raw = t["qkv"].clone()
    go(rotate)
    q, k, v = parts(t)
    q0, k0, v0 = parts({"x": t["x"], "qkv": raw})
    off = t["offsets"].cpu().numpy()
    pos = np.concatenate([off[b] + old["lengths"][b] + np.arange(old["counts"][b]) for b in range(len(off))]).astype(int)
    for new, x, weight in ((q, q0, "q_weight"), (k, k0, "k_weight")):
        y, size = B.rotate(f64(x)[:rows], f64(t[weight]), f64(t["cos"]), f64(t["sin"]), pos, 1e-6, False)
        assert (np.abs(f64(new)[:rows] - y) <= HALF[dt] * np.abs(y) + size * (D / 2 + 12) * U).all()
        assert _torch().equal(new[rows:], x[rows:])
    assert _torch().equal(v, v0)
    go(store)
    c = {"q": q.cpu(), "codes": {}, "scale": {}, "prefix_table": t["prefix_table"].cpu().numpy(), "table": want["page_table"],
         "prefix": t["prefix_lengths"].cpu().numpy(), "members": t["members"].cpu().numpy(), "lengths": want["new_lengths"], "starts": want["starts"], "kind": "e4m3",
         "dt": dt}
    for x, new in (("k", k), ("v", v)):
        c["codes"][x], c["scale"][x] = R.store(f64(new), want["slots"], codes_of(before[x + "_cache"], "e4m3"), before[x + "_scale"].cpu().numpy(), "e4m3")
        assert same_codes(codes_of(t[x + "_cache"], "e4m3"), c["codes"][x], "e4m3") and np.array_equal(t[x + "_scale"].cpu().numpy(), c["scale"][x])
    t["y"].fill_(7.0)
    go(attend)
    prefix_tests.check(c, {"out": t["y"].view(-1, H * G, D)}, prefix_tests.reference(c, 1.0 / np.sqrt(D)), lse=False)
    go(second)
    check_codes(t, "y", "y8")
    go(back)
    check_product(t, "y8", "w_out", t["out"], dt)
    return before


CASES = [([1] * 9, [30, 5, 0, 16, 100, 7, 31, 64, 2], [70, 33], [0, 5, 8]), ([40, 1, 0, 90, 3], [0, 17, 4, 0, 50], [200], [0, 4])]


@pytest.mark.parametrize("case", range(len(CASES)))
def test_step(gpu, case):
    """As one workload: the same results as one operator at a time."""
    t = step_case(gpu, *CASES[case], seed=case)
    before = run_and_check(t)
    after = {k: x.clone() for k, x in t.items()}
    for k, x in before.items():
        t[k].copy_(x)
    t["y"].fill_(7.0)
    prog = go(sequential(*steps(t)))
    assert prog.stats.launches >= 9
    for k, x in after.items():
        assert _torch().equal(t[k].view(_torch().uint8), x.view(_torch().uint8)), k


def test_step_captured(gpu):
    """Captured on a stream of its own and replayed beside eager runs and other work."""
    torch = _torch()
    t = step_case(gpu, *CASES[1], seed=5)
    before = run_and_check(t)
    after = {k: x.clone() for k, x in t.items()}
    prog = sequential(*steps(t)).compile(target="hip_gfx950")

    def restore():
        for k, x in before.items():
            t[k].copy_(x)
        t["y"].fill_(7.0)
        torch.cuda.synchronize()

    def same():
        for k, x in after.items():
            assert torch.equal(t[k].view(torch.uint8), x.view(torch.uint8)), k

    s = torch.cuda.Stream()
    restore()
    with torch.cuda.stream(s):
        prog.execute()
        prog.synchronize()
    same()
    restore()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        prog.execute()
    prog.synchronize()
    for _ in range(3):
        restore()
        g.replay()
        torch.cuda.synchronize()
        same()
        restore()
        prog.execute()
        prog.synchronize()
        same()


def test_two_steps_at_once(gpu):
    """Two programs in flight together, each with a workspace of its own."""
    torch = _torch()
    ts = [step_case(gpu, *CASES[i], seed=7 + i) for i in range(2)]
    befores = [run_and_check(t) for t in ts]
    afters = [{k: x.clone() for k, x in t.items()} for t in ts]
    progs = [sequential(*steps(t)).compile(target="hip_gfx950") for t in ts]
    streams = [torch.cuda.Stream() for _ in ts]
    for _ in range(3):
        for t, before in zip(ts, befores):
            for k, x in before.items():
                t[k].copy_(x)
            t["y"].fill_(7.0)
        torch.cuda.synchronize()
        for p, s in zip(progs, streams):
            with torch.cuda.stream(s):
                p.execute()
        for p in progs:
            p.synchronize()
        for t, after in zip(ts, afters):
            for k, x in after.items():
                assert torch.equal(t[k].view(torch.uint8), x.view(torch.uint8)), k
