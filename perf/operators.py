"""Serving over an 8-bit paged KV cache: the operators that a decode or prefill step runs around its
projections, for timing.

* ``paged_plan``       block tables, slot maps and packed offsets from the requests' lengths;
* ``paged_store``      new keys and values quantised into the 8-bit pages, one scale per page and head;
* ``paged_attention``  causal grouped-query attention of the new tokens over those pages.

``own`` picks between the operators in elementary torch operations and the framework's calls.
"""

import math
import os
import sys

import numpy as np
import torch

own = False

_PKG = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "pto-wsp_amd")

FLOAT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
CODE = {"e4m3": torch.float8_e4m3fn, "i8": torch.int8}
TOP = {"e4m3": 448.0, "i8": 127.0}
TINY = 2.0 ** -126


# ------------------------------------------------------------------------------ cases
def _plan(name, batch, cmin, cmax, lmin, lmax, page):
    return {"name": name, "kind": "plan", "batch": batch, "cmin": cmin, "cmax": cmax, "lmin": lmin, "lmax": lmax, "page": page}


def _store(name, dtype, code, hkv, D, page, batch, cmin, cmax, lmax):
    return {"name": name, "kind": "store", "dtype": dtype, "code": code, "hkv": hkv, "D": D, "page": page, "batch": batch,
            "cmin": cmin, "cmax": cmax, "lmax": lmax}


def _attend(name, dtype, code, hkv, G, D, page, batch, cmin, cmax, lmin, lmax, window=0):
    return {"name": name, "kind": "attend", "dtype": dtype, "code": code, "hkv": hkv, "G": G, "D": D, "page": page,
            "batch": batch, "cmin": cmin, "cmax": cmax, "lmin": lmin, "lmax": lmax, "window": window}


def listed():
    return [
        # One decode step of the benchmark's batch: 64 requests, one token each. Launch latency.
        _plan("plan_decode", 64, 1, 1, 512, 8192, 16),
        # A prefill step: prompts of very different lengths, some of them continued, some idle.
        _plan("plan_prefill", 48, 0, 2048, 0, 4096, 16),
        # Offline generation over many requests at once, prompts and decodes mixed, small pages.
        _plan("plan_many", 4096, 0, 128, 0, 2048, 8),
        # The decode step's new keys and values: 64 tokens into pages that are partly full.
        _store("store_decode", "bf16", "e4m3", 8, 128, 16, 64, 1, 1, 8192),
        # Prompts entering the cache: about 16k tokens.
        _store("store_prefill", "bf16", "e4m3", 8, 128, 16, 16, 1, 2048, 512),
        # Whole-number cache, odd head size and odd pages, 32-bit activations.
        _store("store_odd", "f32", "i8", 3, 80, 24, 21, 0, 300, 100),
        # One chat request with a short context: latency of a single-token call.
        _attend("attend_one", "bf16", "e4m3", 8, 4, 128, 16, 1, 1, 1, 300, 300),
        # The benchmark's paged decode over 8-bit pages: 64 requests of up to 8192 tokens.
        _attend("attend_decode", "bf16", "e4m3", 8, 4, 128, 16, 64, 1, 1, 512, 8192),
        # Two long contexts: few rows, a long axis to split.
        _attend("attend_long", "f16", "i8", 8, 8, 128, 64, 2, 1, 1, 65536, 131072),
        # Odd everything: 7 query heads a key head, head size 80, 8-token pages, 32 bits, a window.
        _attend("attend_odd", "f32", "i8", 2, 7, 80, 8, 37, 1, 3, 1, 5000, 1500),
        # Prompts: every token attends to those before it.
        _attend("attend_prefill", "bf16", "e4m3", 8, 4, 128, 16, 4, 1024, 2048, 1024, 2048),
        # A mixed step: decodes beside chunks of long prompts that are already partly cached.
        _attend("attend_chunks", "bf16", "e4m3", 8, 4, 128, 16, 8, 1, 512, 1024, 6144),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["plan", "store", "store", "attend", "attend", "attend", "attend"])
    page = rng.choice([1, 8, 16, 16, 24, 32, 64, 128])
    if kind == "plan":
        batch = _log_int(rng, 1, 4096)
        cmax = _log_int(rng, 1, max(1, min(8192, (1 << 18) // batch)))
        c = _plan("", batch, rng.choice([0, 1, cmax]), cmax, 0, _log_int(rng, 1, 8192), page)
        c["cmin"] = min(c["cmin"], cmax)
    elif kind == "store":
        hkv, D = rng.choice([1, 2, 3, 4, 8, 16]), rng.choice([16, 64, 80, 96, 128, 128, 192, 256])
        tokens = _log_int(rng, 1, (1 << 24) // (hkv * D))
        batch = min(tokens, _log_int(rng, 1, 512))
        cmax = max(1, tokens // batch)
        c = _store("", rng.choice(["bf16", "bf16", "f16", "f32"]), rng.choice(["e4m3", "e4m3", "i8"]), hkv, D, page, batch,
                   rng.choice([0, 1, cmax]), cmax, _log_int(rng, 1, 4096))
    else:
        hkv, D = rng.choice([1, 2, 4, 8]), rng.choice([16, 64, 64, 80, 96, 128, 128, 128, 256])
        G = rng.choice([1, 2, 4, 5, 7, 8, 16, 24])
        dtype = rng.choice(["bf16", "bf16", "bf16", "f16", "f32"])
        lmax = _log_int(rng, 16, 131072)
        batch = _log_int(rng, 1, 128)
        while batch > 1 and batch * lmax * hkv * D > 3.0e8:
            batch = (batch + 1) // 2
        while batch * lmax * hkv * D > 3.0e8:
            lmax = (lmax + 1) // 2
        cmax = 1
        if rng.random() < 0.5:
            cmax = _log_int(rng, 2, 2048)
            while cmax > 1 and (batch * cmax * G * hkv * lmax > 1.0e9 or batch * cmax * G * hkv * D > 1.0e8):
                cmax = (cmax + 1) // 2
        cmax = min(cmax, lmax)
        lmin = max(cmax, lmax // rng.choice([1, 2, 8, 64]))
        window = rng.choice([0, 0, 0, _log_int(rng, 1, lmax)])
        c = _attend("", dtype, rng.choice(["e4m3", "e4m3", "i8"]), hkv, G, D, page, batch, rng.choice([1, 1, cmax]), cmax, lmin, lmax, window)
    c.pop("name", None)
    return c


# ------------------------------------------------------------------------------ inputs
def _gen(seed):
    g = torch.Generator(device="cuda:0")
    g.manual_seed(seed)
    return g


def _randn(g, shape, dtype=torch.float32):
    return torch.randn(shape, generator=g, device="cuda:0", dtype=torch.float32).to(dtype)


def _ints(x):
    return torch.from_numpy(np.ascontiguousarray(x, dtype=np.int32)).to("cuda:0")


def _requests(case, seed):
    """Per request: tokens held before the step and tokens that the step adds."""
    rng = np.random.default_rng(seed)
    counts = rng.integers(case["cmin"], case["cmax"] + 1, size=case["batch"])
    if case["kind"] == "attend":
        total = rng.integers(case["lmin"], case["lmax"] + 1, size=case["batch"])
        counts = np.minimum(counts, total)
        return total - counts, counts
    return rng.integers(case.get("lmin", 0), case["lmax"] + 1, size=case["batch"]), counts


def _tables(case, seed, held):
    """Pages of `held` tokens per request, in a random order of the pool, and the pages left over:
    enough for one step."""
    page, batch = case["page"], case["batch"]
    pages = -(-held // page)
    order = np.random.default_rng(seed + 1).permutation(int(pages.sum()) + batch * (case["cmax"] // page + 2))
    table = np.zeros((batch, -(-(case["lmax"] + case["cmax"]) // page)), np.int32)
    table[np.arange(table.shape[1])[None] < pages[:, None]] = order[:int(pages.sum())]
    return table, order[int(pages.sum()):]


def _quantised(x, code, dims):
    """Codes of x and their scales, one for each index outside `dims`."""
    scale = (x.abs().amax(dims) / TOP[code]).clamp_min(TINY)
    y = x / scale.reshape([1 if d in dims else s for d, s in enumerate(x.shape)])
    return (y.round() if code == "i8" else y).clamp(-TOP[code], TOP[code]).to(CODE[code]), scale


def _inputs(case, seed):
    """The tensors that a user's program holds before the call."""
    g, kind = _gen(seed), case["kind"]
    before, counts = _requests(case, seed)
    if kind == "plan":
        table, free = _tables(case, seed, before)
        tokens = case["batch"] * case["cmax"]
        return {"lengths": _ints(before), "counts": _ints(counts), "page_table": _ints(table), "free_pages": _ints(free),
                "used": _ints([0]), "new_lengths": _ints(np.zeros(len(counts))), "new_used": _ints([0]),
                "starts": _ints(np.zeros(len(counts) + 1)), "slots": torch.full((tokens,), -2, dtype=torch.int32, device="cuda:0")}
    hkv, D, page, code = (case[k] for k in ("hkv", "D", "page", "code"))
    if kind == "store":
        # Only the last, partly filled page of a request matters to its new tokens.
        before = before % page
        table, free = _tables(case, seed, before)
        pool = case["batch"] * (case["cmax"] // page + 3)
        rows, slots = int(counts.sum()), []
        for b, n in enumerate(counts):
            pos = before[b] + np.arange(n)
            full = np.concatenate([table[b, :-(-before[b] // page)], free[b * (case["cmax"] // page + 2):]])
            slots.append(full[pos // page].astype(np.int64) * page + pos % page)
        pad = case["batch"] * case["cmax"]  # a step's buffers are as long as its largest batch
        slots = np.concatenate(slots + [np.full(pad - rows, -1)])
        dt = FLOAT[case["dtype"]]
        heads = torch.exp2(_randn(g, (hkv, 1)))
        t = {"k": (_randn(g, (pad, hkv, D)) * heads).to(dt), "v": _randn(g, (pad, hkv, D), dt), "slots": _ints(slots)}
        for x in ("k", "v"):
            t[x + "_cache"], t[x + "_scale"] = _quantised(_randn(g, (pool, hkv, page, D)), code, (2, 3))
        return t
    total = before + counts
    table, _ = _tables(case, seed, total)
    pool = int(table.max()) + 1
    rows = case["batch"] * case["cmax"]
    t = {"q": _randn(g, (rows, hkv * case["G"], D), FLOAT[case["dtype"]]), "page_table": _ints(table), "lengths": _ints(total),
         "starts": _ints(np.concatenate([[0], np.cumsum(counts)]))}
    for x in ("k", "v"):
        # Keys and values of a page share a scale; pages and heads differ in theirs.
        codes, _ = _quantised(_randn(g, (pool, hkv, page, D)), code, (2, 3))
        t[x + "_cache"] = codes
        t[x + "_scale"] = torch.exp2(0.5 * _randn(g, (pool, hkv))) * (3.5 / TOP[code])
    t["out"] = torch.zeros_like(t["q"])
    return t


# ------------------------------------------------------------------------------ the framework's calls
def _program(case, t):
    if _PKG not in sys.path:
        sys.path.insert(0, _PKG)
    from pto_wsp import DType, Tensor, paged_attention, paged_plan, paged_store

    kinds = {torch.float32: DType.F32, torch.float16: DType.F16, torch.bfloat16: DType.BF16, torch.int32: DType.I32,
             torch.int8: DType.I8, torch.float8_e4m3fn: DType.F8E4M3}
    T = {name: Tensor(data=x, shape=tuple(x.shape), dtype=kinds[x.dtype]) for name, x in t.items()}
    if case["kind"] == "plan":
        return paged_plan(**T, page_size=case["page"]).compile(target="hip_gfx950")
    if case["kind"] == "store":
        return paged_store(**T).compile(target="hip_gfx950")
    return paged_attention(**T, scale=1.0 / math.sqrt(case["D"]), window=case["window"]).compile(target="hip_gfx950")


def prepare(case, seed):
    t = _inputs(case, seed)
    state = {"case": case, "t": t}
    if own:
        state["program"] = _program(case, t)
    return state


OUTPUTS = {"plan": ("page_table", "new_lengths", "new_used", "starts", "slots"), "store": ("k_cache", "v_cache", "k_scale", "v_scale"),
           "attend": ("out",)}


def run(state):
    case, t = state["case"], state["t"]
    if own:
        state["program"].execute()
        state["program"].synchronize()
    else:
        {"plan": _plain_plan, "store": _plain_store, "attend": _plain_attend}[case["kind"]](case, t)
    return {k: t[k] for k in OUTPUTS[case["kind"]]}


# ------------------------------------------------------------------------------ plain forms
def _plain_plan(case, t):
    page, lengths, counts, table, slots = case["page"], t["lengths"], t["counts"], t["page_table"], t["slots"]
    total = lengths + counts
    old, new = (lengths + page - 1) // page, (total + page - 1) // page
    first = t["used"] + torch.cumsum(new - old, 0, dtype=torch.int32) - (new - old)
    j = torch.arange(table.shape[1], device=table.device)[None]
    fresh = (j >= old[:, None]) & (j < new[:, None])
    took = t["free_pages"][(first[:, None] + j - old[:, None]).clamp(0, max(0, len(t["free_pages"]) - 1))]
    table.copy_(torch.where(fresh, took, table))
    t["new_lengths"].copy_(total)
    t["new_used"].copy_(t["used"] + (new - old).sum())
    t["starts"][:1] = 0
    t["starts"][1:] = torch.cumsum(counts, 0)
    row = torch.arange(len(slots), dtype=torch.int32, device=slots.device)
    seq = torch.searchsorted(t["starts"][1:].contiguous(), row, right=True).clamp_max(len(counts) - 1)
    pos = lengths[seq] + row - t["starts"][seq]
    p = table[seq, (pos // page).clamp(0, table.shape[1] - 1)]
    slots.copy_(torch.where(row < t["starts"][-1], p * page + pos % page, -1))


def _plain_store(case, t):
    page, top, code = case["page"], TOP[case["code"]], CODE[case["code"]]
    row = torch.nonzero(t["slots"] >= 0)[:, 0]
    slot = t["slots"][row].long()
    if not len(row):
        return
    touched, where = torch.unique(slot // page, return_inverse=True)
    off = slot % page
    # Tokens ahead of the first new one of a page stay in it.
    low = torch.full((len(touched),), page, device=off.device).scatter_reduce_(0, where, off, "amin")
    kept = torch.arange(page, device=off.device)[None] < low[:, None]
    for x in ("k", "v"):
        cache, scales = t[x + "_cache"], t[x + "_scale"]
        new = t[x][row].float()
        most = torch.zeros((len(touched), new.shape[1]), device=new.device)
        most.scatter_reduce_(0, where[:, None].expand(-1, new.shape[1]), new.abs().amax(-1), "amax")
        old = torch.where(low[:, None] > 0, scales[touched], 0.0)
        scale = torch.maximum((most / torch.full_like(most, top)).clamp_min(TINY), old)
        inverse = 1.0 / scale
        codes = cache.view(torch.int8)[touched].view(code)
        y = codes.float() * old[:, :, None, None] * inverse[:, :, None, None]
        y = (y.round() if code == torch.int8 else y).clamp(-top, top).to(code)
        grown = (scale > old)[:, :, None, None] & kept[:, None, :, None]
        codes = torch.where(grown, y.view(torch.int8), codes.view(torch.int8))
        z = new * inverse[where][:, :, None]
        codes[where, :, off] = (z.round() if code == torch.int8 else z).clamp(-top, top).to(code).view(torch.int8)
        cache.view(torch.int8)[touched] = codes
        scales[touched] = scale


def _plain_attend(case, t):
    hkv, G, D, page, window = (case[k] for k in ("hkv", "G", "D", "page", "window"))
    starts, lengths, table = t["starts"].long(), t["lengths"].long(), t["page_table"].long()
    counts = starts[1:] - starts[:-1]
    most, longest, batch = case["cmax"], table.shape[1] * page, len(lengths)
    tok = torch.arange(longest, device=table.device)

    def gathered(x):
        pages = table[:, tok // page]  # [batch, tokens]
        codes = t[x + "_cache"].view(torch.int8)[pages, :, tok % page].view(CODE[case["code"]])
        return (codes.float() * t[x + "_scale"][pages][..., None]).permute(0, 2, 1, 3)  # [batch, head, token, D]

    i = torch.arange(most, device=table.device)
    rows = (starts[:-1, None] + i).clamp_max(len(t["q"]) - 1)
    q = t["q"][rows].float().reshape(batch, most, hkv, G, D).permute(0, 2, 1, 3, 4).reshape(batch, hkv, most * G, D)
    s = torch.matmul(q, gathered("k").transpose(2, 3)) * (1.0 / math.sqrt(D))
    pos = (lengths - counts)[:, None] + i  # [batch, query]
    seen = (tok <= pos[..., None]) & (tok < lengths[:, None, None])
    if window:
        seen &= tok > pos[..., None] - window
    seen = seen[:, None, :, None].expand(batch, 1, most, G, longest).reshape(batch, 1, most * G, longest)
    s = torch.where(seen, s, -math.inf)
    e = torch.exp(s - s.amax(-1, keepdim=True).clamp_min(-3.0e38))
    del s, seen
    o = torch.matmul(e, gathered("v")) / e.sum(-1, keepdim=True)
    o = o.reshape(batch, hkv, most, G, D).permute(0, 2, 1, 3, 4).reshape(batch * most, hkv * G, D)
    take = torch.nonzero((i < counts[:, None]).reshape(-1))[:, 0]
    t["out"][:len(take)] = o[take].to(t["out"].dtype)  # rows behind the last request stay as they were


# ------------------------------------------------------------------------------ work and accuracy
def work(case):
    kind, batch, page = case["kind"], case["batch"], case["page"]
    new = batch * (case["cmin"] + case["cmax"]) / 2.0
    if kind == "plan":
        # Lengths and counts in and out, the page of every token, one slot per row of the buffer.
        pages = new / page + batch
        return {"bytes": 4 * (4 * batch + 2 * pages + batch * case["cmax"]), "flops": 4 * batch * case["cmax"]}
    hkv, D = case["hkv"], case["D"]
    size = torch.finfo(FLOAT[case["dtype"]]).bits // 8
    if kind == "store":
        # New keys and values in, their codes out, one scale per page that they touch, the slots.
        return {"bytes": 2 * new * hkv * D * (size + 1) + 8 * hkv * (new / page + batch) + 4 * new, "flops": 8 * new * hkv * D}
    mean = (case["lmin"] + case["lmax"]) / 2.0
    count = min(new / batch, mean)
    seen = max(1.0, mean - (count - 1) / 2.0)  # keys of an average new token
    held = mean
    if case["window"]:
        seen, held = min(seen, case["window"]), min(mean, case["window"] + count - 1)
    return {"bytes": batch * (2 * held * hkv * D + held / page * (4 + 8 * hkv)) + 2 * new * hkv * case["G"] * D * size,
            "flops": 4 * new * hkv * case["G"] * D * seen}


def _nearest(x):
    """The float32 value nearest to x, in 64 bits."""
    return x.to(torch.float32).double()


def _exact_store(case, t):
    """Page by page. A scale, its reciprocal and a quotient are each the float32 value nearest to
    the exact one; codes are the nearest of their type."""
    page, top, whole = case["page"], TOP[case["code"]], case["code"] == "i8"
    slots = t["slots"].cpu().numpy()
    pages = {}
    for r, s in enumerate(slots):
        if s >= 0:
            pages.setdefault(int(s) // page, []).append((r, int(s) % page))
    out = {}
    for x in ("k", "v"):
        values, scales = t[x + "_cache"].double(), t[x + "_scale"].double()

        def coded(y):
            y = _nearest(y).clamp(-top, top)
            return y.round() if whole else y.to(torch.float32).to(torch.float8_e4m3fn).double()

        for p, rows in pages.items():
            r, off = torch.tensor([a for a, _ in rows], device=values.device), torch.tensor([b for _, b in rows], device=values.device)
            low = min(b for _, b in rows)
            new = t[x][r].double()
            scale = _nearest(new.abs().amax((0, 2)) / top).clamp_min(TINY)
            if low:
                scale = torch.maximum(scale, scales[p])
            inverse = _nearest(1.0 / scale)
            if low:
                grown = (scale > scales[p])[:, None, None]
                values[p, :, :low] = torch.where(grown, coded(_nearest(values[p, :, :low] * scales[p][:, None, None]) * inverse[:, None, None]),
                                                 values[p, :, :low])
            values[p, :, off] = coded(new * inverse[:, None]).transpose(0, 1)
            scales[p] = scale
        out[x + "_cache"] = values.to(torch.int8) if whole else values
        out[x + "_scale"] = scales
    return {k: out[k] for k in OUTPUTS["store"]}


def _exact_attend(case, t):
    hkv, G, D, page, window = (case[k] for k in ("hkv", "G", "D", "page", "window"))
    starts, lengths = t["starts"].tolist(), t["lengths"].tolist()
    out = torch.zeros(t["out"].shape, dtype=torch.float64, device=t["out"].device)
    for b, total in enumerate(lengths):
        n = starts[b + 1] - starts[b]
        if not n:
            continue
        pages = t["page_table"][b, :-(-total // page)].long()
        low = max(0, total - n + 1 - window) if window else 0
        for h in range(hkv):
            k, v = ((t[x + "_cache"][pages, h].double() * t[x + "_scale"][pages, h].double()[:, None, None]).reshape(-1, D)[low:total] for x in "kv")
            at = low + torch.arange(len(k), device=k.device)
            for lo in range(0, n, 512):
                hi = min(n, lo + 512)
                q = t["q"][starts[b] + lo:starts[b] + hi, h * G:(h + 1) * G].double()
                s = (q.reshape(-1, D) @ k.T.contiguous() / math.sqrt(D)).reshape(hi - lo, G, -1)
                pos = (total - n + torch.arange(lo, hi, device=k.device))[:, None, None]
                s = s.masked_fill((at > pos) | (at <= pos - window if window else at < 0), -math.inf)
                out[starts[b] + lo:starts[b] + hi, h * G:(h + 1) * G] = (torch.softmax(s, -1).reshape(-1, len(k)) @ v).reshape(hi - lo, G, D)
    return {"out": out}


def exact(case, seed):
    if case["kind"] == "plan":
        return None  # whole numbers
    t = _inputs(case, seed)
    return _exact_store(case, t) if case["kind"] == "store" else _exact_attend(case, t)
