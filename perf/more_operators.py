"""A serving step around the 8-bit paged KV cache: the operators between its projections and its attention,
for timing.

* ``block_quantize``          activations or weights in e4m3, a scale for each block of 128 columns;
* ``block_matmul``            their product;
* ``paged_norm_rotate``       norms of queries and keys a head, and their rotation by position;
* ``paged_prefix_attention``  attention of requests that share a prefix, which is read once for all of them.

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
BLOCK = 128


# ------------------------------------------------------------------------------ cases
def _quantize(name, dtype, M, K, rows=1):
    return {"name": name, "kind": "quantize", "dtype": dtype, "M": M, "K": K, "rows": rows}


def _matmul(name, dtype, M, N, K):
    return {"name": name, "kind": "matmul", "dtype": dtype, "M": M, "N": N, "K": K}


def _rotate(name, dtype, hkv, G, D, R, interleaved, norm, batch, cmin, cmax, lmax, prefix):
    return {"name": name, "kind": "rotate", "dtype": dtype, "hkv": hkv, "G": G, "D": D, "R": R, "interleaved": interleaved,
            "norm": norm, "batch": batch, "cmin": cmin, "cmax": cmax, "lmax": lmax, "prefix": prefix}


def _prefix(name, dtype, code, hkv, G, D, page, groups, batch, loose, cmin, cmax, lmin, lmax, pmin, pmax):
    return {"name": name, "kind": "prefix", "dtype": dtype, "code": code, "hkv": hkv, "G": G, "D": D, "page": page,
            "groups": groups, "batch": batch, "loose": loose, "cmin": cmin, "cmax": cmax, "lmin": lmin, "lmax": lmax,
            "pmin": pmin, "pmax": pmax}


def listed():
    return [
        # Activations of a decode step of 64 requests ahead of a projection. Launch latency.
        _quantize("quantize_decode", "bf16", 64, 4096),
        # Activations of 16384 prompt tokens.
        _quantize("quantize_prefill", "bf16", 16384, 4096),
        # The projection to 32 query and 2 x 8 key heads of 128 in a decode step: the weights are the work.
        _matmul("matmul_decode", "bf16", 64, 6144, 4096),
        # The same for 8192 prompt tokens.
        _matmul("matmul_prefill", "bf16", 8192, 6144, 4096),
        # Odd everything: rows, columns and a depth that no vector load divides, 32-bit results.
        _matmul("matmul_odd", "f32", 300, 1000, 1160),
        # One token of each of 64 requests, the whole head rotated, halves paired.
        _rotate("rotate_decode", "bf16", 8, 4, 128, 128, False, True, 64, 1, 1, 8192, 0),
        # Prompts entering the cache: about 16k tokens.
        _rotate("rotate_prefill", "bf16", 8, 4, 128, 128, False, True, 16, 1, 2048, 512, 0),
        # Odd heads of 32 bits of which 32 dims turn, neighbours paired, tokens behind a prefix.
        _rotate("rotate_odd", "f32", 3, 5, 80, 32, True, True, 21, 0, 300, 100, 700),
        # Four chats that begin with the same instructions. Latency.
        _prefix("prefix_few", "bf16", "e4m3", 8, 4, 128, 16, 1, 4, 0, 1, 1, 1, 100, 900, 1000),
        # The benchmark's decode batch behind one long document.
        _prefix("prefix_decode", "bf16", "e4m3", 8, 4, 128, 16, 1, 64, 0, 1, 1, 64, 1024, 16384, 16384),
        # Three instructions among the requests and some without: odd heads, 8-token pages, 32 bits.
        _prefix("prefix_groups", "f32", "i8", 2, 7, 80, 8, 3, 37, 5, 0, 3, 3, 300, 200, 5000),
        # Questions about one document: prompts behind a prefix.
        _prefix("prefix_prompts", "bf16", "e4m3", 8, 4, 128, 16, 2, 16, 2, 1, 256, 256, 512, 2048, 8192),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _depth(rng, most):
    """Columns: whole blocks, whole vectors, or any number."""
    K = _log_int(rng, 1, most)
    step = rng.choice([128, 128, 16, 1])
    return max(1, K // step * step)


def draw(rng):
    kind = rng.choice(["quantize", "matmul", "matmul", "rotate", "prefix", "prefix"])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    if kind == "quantize":
        K = _depth(rng, 16384)
        # 16384 x 4096 elements of 2 bytes at most
        c = _quantize("", dtype, _log_int(rng, 1, (1 << 26) // K // (2 if dtype == "f32" else 1)), K, rng.choice([1, 1, 128]))
    elif kind == "matmul":
        K, N = _depth(rng, 16384), _log_int(rng, 1, 16384)
        M = _log_int(rng, 1, 16384)
        if rng.random() < 0.6:
            N = max(1, N // 128 * 128)
        while M * N * K > 8192 * 6144 * 4096:
            M = (M + 1) // 2
        c = _matmul("", dtype, M, N, K)
    elif kind == "rotate":
        hkv, G = rng.choice([1, 2, 3, 4, 8]), rng.choice([1, 2, 4, 5, 7, 8])
        D = rng.choice([16, 64, 80, 96, 128, 128, 192, 256])
        tokens = _log_int(rng, 1, (1 << 25) // (hkv * (G + 1) * D))
        batch = min(tokens, _log_int(rng, 1, 512))
        cmax = max(1, tokens // batch)
        c = _rotate("", dtype, hkv, G, D, rng.choice([D, D, D // 2, 2 * rng.randint(1, D // 2)]), rng.random() < 0.3,
                    rng.random() < 0.8, batch, rng.choice([0, 1, cmax]), cmax, _log_int(rng, 1, 16384), rng.choice([0, _log_int(rng, 1, 4096)]))
    else:
        hkv, D = rng.choice([1, 2, 4, 8]), rng.choice([16, 64, 64, 80, 96, 128, 128, 128, 256])
        G = rng.choice([1, 2, 4, 5, 7, 8, 16, 24])
        page = rng.choice([1, 8, 16, 16, 24, 32, 64, 128])
        pmax, batch = _log_int(rng, 16, 32768), _log_int(rng, 2, 128)
        groups = rng.choice([1, 1, 2, min(batch, 5)])
        lmax = _log_int(rng, 1, 4096)
        cmax = 1 if rng.random() < 0.6 else _log_int(rng, 1, 512)
        cmax = min(cmax, lmax)
        while batch > groups and batch * cmax * G * hkv * (pmax + lmax) > 5.0e8:
            batch -= (batch - groups + 1) // 2
        while cmax > 1 and batch * cmax * G * hkv * (pmax + lmax) > 5.0e8:
            cmax = (cmax + 1) // 2
        while batch * lmax * hkv * D + groups * pmax * hkv * D > 6.0e7:
            lmax, pmax = max(cmax, lmax // 2), max(1, pmax // 2)
        lmin = max(cmax, lmax // rng.choice([1, 2, 8, 64]))
        c = _prefix("", dtype, rng.choice(["e4m3", "e4m3", "i8"]), hkv, G, D, page, groups, batch, rng.randint(0, batch - groups) // 2,
                    rng.choice([0, 1, cmax]), cmax, lmin, lmax, max(1, pmax // rng.choice([1, 2, 64])), pmax)
        c["cmin"] = min(c["cmin"], cmax)
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


def _blocks(n):
    return -(-n // BLOCK)


def _activations(g, M, K, dtype=torch.float32):
    """Rows whose columns differ in size, as a model's channels do."""
    return (_randn(g, (M, K)) * torch.exp2(_randn(g, (K,)))).to(dtype)


def _codes_of_weights(g, N, K):
    """e4m3 codes of random weights and the scales of their 128 x 128 blocks."""
    w = _randn(g, (N, K)) * 0.02
    padded = torch.zeros((_blocks(N) * BLOCK, _blocks(K) * BLOCK), device=w.device)
    padded[:N, :K] = w
    scale = (padded.reshape(_blocks(N), BLOCK, _blocks(K), BLOCK).abs().amax((1, 3)) / 448.0).clamp_min(TINY)
    codes = (w / scale.repeat_interleave(BLOCK, 0)[:N].repeat_interleave(BLOCK, 1)[:, :K]).clamp(-448.0, 448.0)
    return codes.to(torch.float8_e4m3fn), scale


def _counts(case, seed):
    return np.random.default_rng(seed).integers(case["cmin"], case["cmax"] + 1, size=case["batch"])


def _rotate_inputs(case, g, seed):
    rng = np.random.default_rng(seed + 1)
    counts = _counts(case, seed)
    lengths = counts + rng.integers(0, case["lmax"] + 1, size=case["batch"])
    offsets = rng.integers(0, case["prefix"] + 1, size=case["batch"])
    hkv, G, D, R, dt = case["hkv"], case["G"], case["D"], case["R"], FLOAT[case["dtype"]]
    rows = case["batch"] * case["cmax"]  # a step's buffers are as long as its largest batch
    # Queries, keys and values of a row lie one behind the other, as the projection leaves them.
    packed = _randn(g, (rows, hkv * (G + 2), D), dt)
    most = case["lmax"] + case["cmax"] + case["prefix"] + 1
    angles = torch.arange(most, device="cuda:0", dtype=torch.float64)[:, None] * torch.pow(
        10000.0, -torch.arange(0, R, 2, device="cuda:0", dtype=torch.float64) / R)
    t = {"q": packed[:, :hkv * G], "k": packed[:, hkv * G:hkv * (G + 1)], "cos": torch.cos(angles).float(), "sin": torch.sin(angles).float(),
         "lengths": _ints(lengths), "starts": _ints(np.concatenate([[0], np.cumsum(counts)])),
         "q_out": torch.zeros((rows, hkv * G, D), dtype=dt, device="cuda:0"), "k_out": torch.zeros((rows, hkv, D), dtype=dt, device="cuda:0")}
    if case["prefix"]:
        t["offsets"] = _ints(offsets)
    if case["norm"]:
        t["q_weight"], t["k_weight"] = (1.0 + 0.2 * _randn(g, (D,))).to(dt), (1.0 + 0.2 * _randn(g, (D,))).to(dt)
    return t, None


def _prefix_inputs(case, g, seed):
    rng = np.random.default_rng(seed + 1)
    page, batch, groups = case["page"], case["batch"], case["groups"]
    lengths = rng.integers(case["lmin"], case["lmax"] + 1, size=batch)
    counts = np.minimum(_counts(case, seed), lengths)
    prefix = rng.integers(case["pmin"], case["pmax"] + 1, size=groups)
    # The requests of a group follow each other; the last ones have no prefix.
    inner = np.sort(rng.choice(np.arange(1, batch - case["loose"]), groups - 1, replace=False)) if groups > 1 else np.zeros(0, np.int64)
    members = np.concatenate([[0], inner, [batch - case["loose"]]]).astype(np.int64)
    pages, ppages = -(-lengths // page), -(-prefix // page)
    order = rng.permutation(int(pages.sum() + ppages.sum()))
    table, ptable = np.zeros((batch, -(-case["lmax"] // page)), np.int32), np.zeros((groups, -(-case["pmax"] // page)), np.int32)
    table[np.arange(table.shape[1])[None] < pages[:, None]] = order[:int(pages.sum())]
    ptable[np.arange(ptable.shape[1])[None] < ppages[:, None]] = order[int(pages.sum()):]
    hkv, D, code = case["hkv"], case["D"], case["code"]
    starts = np.concatenate([[0], np.cumsum(counts)])
    t = {"q": _randn(g, (batch * case["cmax"], hkv * case["G"], D), FLOAT[case["dtype"]]), "prefix_table": _ints(ptable),
         "prefix_lengths": _ints(prefix), "members": _ints(members), "page_table": _ints(table), "lengths": _ints(lengths), "starts": _ints(starts)}
    for x in ("k", "v"):
        # Keys and values of a page share a scale; pages and heads differ in theirs.
        y = _randn(g, (len(order), hkv, page, D))
        y = y * (TOP[code] / y.abs().amax((2, 3), keepdim=True))
        t[x + "_cache"] = (y.round() if code == "i8" else y).clamp(-TOP[code], TOP[code]).to(CODE[code])
        t[x + "_scale"] = torch.exp2(0.5 * _randn(g, (len(order), hkv))) * (3.5 / TOP[code])
    t["out"] = torch.zeros_like(t["q"])
    # What the scheduler that made the batch knows of it.
    return t, {"rows": [int(starts[m]) for m in members], "prefix": [int(n) for n in prefix]}


def _inputs(case, seed):
    """The tensors that a user's program holds before the call, and what it knows of them on the host."""
    g, kind = _gen(seed), case["kind"]
    if kind == "quantize":
        M, K = case["M"], case["K"]
        return {"x": _activations(g, M, K, FLOAT[case["dtype"]]), "codes": torch.zeros((M, K), device="cuda:0").to(torch.float8_e4m3fn),
                "scales": torch.zeros((-(-M // case["rows"]), _blocks(K)), device="cuda:0")}, None
    if kind == "matmul":
        M, N, K = case["M"], case["N"], case["K"]
        t = dict(zip(("a", "a_scale"), _plain_quantize(_activations(g, M, K), 1)))
        t["b"], t["b_scale"] = _codes_of_weights(g, N, K)
        t["out"] = torch.zeros((M, N), dtype=FLOAT[case["dtype"]], device="cuda:0")
        return t, None
    return _rotate_inputs(case, g, seed) if kind == "rotate" else _prefix_inputs(case, g, seed)


# ------------------------------------------------------------------------------ the framework's calls
def _program(case, t):
    if _PKG not in sys.path:
        sys.path.insert(0, _PKG)
    from pto_wsp import DType, Tensor, block_matmul, block_quantize, paged_norm_rotate, paged_prefix_attention

    kinds = {torch.float32: DType.F32, torch.float16: DType.F16, torch.bfloat16: DType.BF16, torch.int32: DType.I32,
             torch.int8: DType.I8, torch.float8_e4m3fn: DType.F8E4M3}
    T = {name: Tensor(data=x, shape=tuple(x.shape), dtype=kinds[x.dtype]) for name, x in t.items()}
    if case["kind"] == "quantize":
        w = block_quantize(**T, rows=case["rows"])
    elif case["kind"] == "matmul":
        w = block_matmul(**T)
    elif case["kind"] == "rotate":
        w = paged_norm_rotate(**T, eps=1e-6, interleaved=case["interleaved"])
    else:
        w = paged_prefix_attention(**T, scale=1.0 / math.sqrt(case["D"]))
    return w.compile(target="hip_gfx950")


def prepare(case, seed):
    t, plan = _inputs(case, seed)
    state = {"case": case, "t": t, "plan": plan}
    if own:
        state["program"] = _program(case, t)
    return state


OUTPUTS = {"quantize": ("codes", "scales"), "matmul": ("out",), "rotate": ("q_out", "k_out"), "prefix": ("out",)}


def run(state):
    case, t = state["case"], state["t"]
    if own:
        state["program"].execute()
        state["program"].synchronize()
    elif case["kind"] == "quantize":
        codes, scales = _plain_quantize(t["x"], case["rows"])
        t["codes"].view(torch.int8).copy_(codes.view(torch.int8))
        t["scales"].copy_(scales)
    else:
        {"matmul": _plain_matmul, "rotate": _plain_rotate, "prefix": _plain_prefix}[case["kind"]](case, t, state["plan"])
    return {k: t[k] for k in OUTPUTS[case["kind"]]}


# ------------------------------------------------------------------------------ plain forms
def _plain_quantize(x, rows):
    M, K = x.shape
    most = torch.zeros((-(-M // rows) * rows, _blocks(K) * BLOCK), device=x.device)
    most[:M, :K] = x.float().abs()
    most = most.reshape(-1, rows, _blocks(K), BLOCK).amax((1, 3))
    scale = (most / torch.full_like(most, 448.0)).clamp_min(TINY)
    inverse = (1.0 / scale).repeat_interleave(rows, 0)[:M].repeat_interleave(BLOCK, 1)[:, :K]
    return (x.float() * inverse).clamp(-448.0, 448.0).to(torch.float8_e4m3fn), scale


def _plain_matmul(case, t, plan):
    a = t["a"].float() * t["a_scale"].repeat_interleave(BLOCK, 1)[:, :case["K"]]
    b = t["b"].float() * t["b_scale"].repeat_interleave(BLOCK, 0)[:case["N"]].repeat_interleave(BLOCK, 1)[:, :case["K"]]
    t["out"].copy_(torch.matmul(a, b.t()))


def _plain_rotate(case, t, plan):
    R, rows = case["R"], len(t["q"])
    starts, lengths = t["starts"].long(), t["lengths"].long()
    row = torch.arange(rows, device=starts.device)
    seq = torch.searchsorted(starts[1:].contiguous(), row, right=True).clamp_max(len(lengths) - 1)
    pos = lengths[seq] - starts[seq + 1] + row
    if "offsets" in t:
        pos = pos + t["offsets"].long()[seq]
    real = row < starts[-1]
    pos = pos.clamp(0, len(t["cos"]) - 1)
    c, s = t["cos"][pos][:, None], t["sin"][pos][:, None]
    for x in ("q", "k"):
        y = t[x].float()
        if x + "_weight" in t:
            y = y * torch.rsqrt((y * y).mean(-1, keepdim=True) + 1e-6) * t[x + "_weight"].float()
        lo, hi = (slice(0, R, 2), slice(1, R, 2)) if case["interleaved"] else (slice(0, R // 2), slice(R // 2, R))
        z = y.clone()
        z[..., lo] = y[..., lo] * c - y[..., hi] * s
        z[..., hi] = y[..., hi] * c + y[..., lo] * s
        t[x + "_out"].copy_(torch.where(real[:, None, None], z.to(t[x].dtype), t[x + "_out"]))  # rows behind the last request stay


def _paged(case, t, x, pages, tok):
    """Keys or values of the tokens `tok` of the tables `pages`, [..., tokens, head, D]."""
    page = case["page"]
    at = pages[..., tok // page]
    codes = t[x + "_cache"].view(torch.int8)[at, :, tok % page].view(CODE[case["code"]])
    return codes.float() * t[x + "_scale"][at][..., None]


def _plain_prefix(case, t, plan):
    hkv, G, D, scale = case["hkv"], case["G"], case["D"], 1.0 / math.sqrt(case["D"])
    starts, lengths, table = t["starts"].long(), t["lengths"].long(), t["page_table"].long()
    counts = starts[1:] - starts[:-1]
    most, longest, batch = case["cmax"], int(table.shape[1]) * case["page"], len(lengths)
    tok = torch.arange(longest, device=table.device)
    # Each request's rows over its own tokens.
    i = torch.arange(most, device=table.device)
    rows = (starts[:-1, None] + i).clamp_max(len(t["q"]) - 1)
    q = t["q"][rows].float().reshape(batch, most, hkv, G, D).permute(0, 2, 1, 3, 4).reshape(batch, hkv, most * G, D)
    s = torch.matmul(q, _paged(case, t, "k", table, tok).permute(0, 2, 3, 1).contiguous()) * scale
    pos = (lengths - counts)[:, None] + i
    seen = ((tok <= pos[..., None]) & (tok < lengths[:, None, None]))[:, None, :, None]
    s = torch.where(seen.expand(batch, 1, most, G, longest).reshape(batch, 1, most * G, longest), s, -math.inf)
    top = s.amax(-1, keepdim=True)
    e = torch.exp(s - top.clamp_min(-3.0e38))
    del s, seen
    o = torch.matmul(e, _paged(case, t, "v", table, tok).permute(0, 2, 1, 3).contiguous())
    o = torch.cat([o, e.sum(-1, keepdim=True), top], -1)
    del e
    take = torch.nonzero((i < counts[:, None]).reshape(-1))[:, 0]
    o = o.reshape(batch, hkv, most, G, D + 2).permute(0, 2, 1, 3, 4).reshape(batch * most, hkv, G, D + 2)[take]
    o, total, top = o[..., :D], o[..., D], o[..., D + 1]
    # The rows of a group over its prefix, joined with those.
    for g, (r0, r1, n) in enumerate(zip(plan["rows"], plan["rows"][1:], plan["prefix"])):
        if r0 == r1:
            continue
        tok = torch.arange(n, device=table.device)
        pages = t["prefix_table"][g].long()
        q = t["q"][r0:r1].float().reshape(r1 - r0, hkv, G, D).transpose(0, 1).reshape(hkv, (r1 - r0) * G, D)
        s = torch.matmul(q, _paged(case, t, "k", pages, tok).permute(1, 2, 0).contiguous()) * scale
        peak = s.amax(-1, keepdim=True)
        e = torch.exp(s - peak)
        del s
        p = torch.matmul(e, _paged(case, t, "v", pages, tok).permute(1, 0, 2).contiguous())
        p = torch.cat([p, e.sum(-1, keepdim=True), peak], -1).reshape(hkv, r1 - r0, G, D + 2).transpose(0, 1)
        del e
        both = torch.maximum(top[r0:r1], p[..., D + 1])
        mine, theirs = torch.exp(top[r0:r1] - both), torch.exp(p[..., D + 1] - both)
        o[r0:r1] = o[r0:r1] * mine[..., None] + p[..., :D] * theirs[..., None]
        total[r0:r1] = total[r0:r1] * mine + p[..., D] * theirs
    t["out"][:len(o)] = (o / total[..., None]).reshape(-1, hkv * G, D).to(t["out"].dtype)  # rows behind the last request stay


# ------------------------------------------------------------------------------ work and accuracy
def work(case):
    kind = case["kind"]
    size = torch.finfo(FLOAT[case["dtype"]]).bits // 8
    if kind == "quantize":
        # Numbers in, codes and scales out.
        M, K = case["M"], case["K"]
        return {"bytes": M * K * (size + 1) + 4 * _blocks(K) * -(-M // case["rows"]), "flops": 3 * M * K}
    if kind == "matmul":
        M, N, K = case["M"], case["N"], case["K"]
        return {"bytes": (M + N) * K + M * N * size + 4 * _blocks(K) * (M + _blocks(N)), "flops": 2 * M * N * K}
    batch, hkv, G, D = (case[k] for k in ("batch", "hkv", "G", "D"))
    mean = (case["cmin"] + case["cmax"]) / 2.0
    new = batch * mean
    if kind == "rotate":
        # Queries and keys in and out, a row of the tables for each token at most once.
        return {"bytes": new * (2 * hkv * (G + 1) * D * size + 4 * case["R"]), "flops": new * hkv * (G + 1) * (4 * D + 3 * case["R"])}
    held, prefix = (case["lmin"] + case["lmax"]) / 2.0, (case["pmin"] + case["pmax"]) / 2.0
    seen = max(1.0, held - (mean - 1) / 2.0)  # own keys of an average new token
    behind = new * (batch - case["loose"]) / batch  # rows that see a prefix
    tokens = batch * held + case["groups"] * prefix
    return {"bytes": tokens * (2 * hkv * D + (4 + 8 * hkv) / case["page"]) + 2 * new * hkv * G * D * size,
            "flops": 4 * hkv * G * D * (new * seen + behind * prefix)}


def _nearest(x):
    """The float32 value nearest to x, in 64 bits."""
    return x.to(torch.float32).double()


def _exact_quantize(case, t):
    """A scale and its reciprocal are each the float32 value nearest to the exact one, as is a quotient; codes are the nearest of
    their type."""
    x, rows = t["x"].double(), case["rows"]
    codes, scales = torch.empty_like(x), torch.empty(t["scales"].shape, dtype=torch.float64, device=x.device)
    for j in range(scales.shape[1]):
        part = x[:, BLOCK * j:BLOCK * (j + 1)]
        most = part.abs().amax(1)
        if rows > 1:
            pad = torch.zeros(len(scales) * rows, dtype=torch.float64, device=x.device)
            pad[:len(most)] = most
            most = pad.reshape(-1, rows).amax(1)
        scales[:, j] = _nearest(most / 448.0).clamp_min(TINY)
        inverse = _nearest(1.0 / scales[:, j]).repeat_interleave(rows)[:len(x), None]
        codes[:, BLOCK * j:BLOCK * (j + 1)] = (part * inverse).to(torch.float32).clamp(-448.0, 448.0).to(torch.float8_e4m3fn).double()
    return {"codes": codes, "scales": scales}


def _exact_matmul(case, t):
    out = torch.zeros(t["out"].shape, dtype=torch.float64, device=t["out"].device)
    a, b = t["a"].double(), t["b"].double()
    for j in range(_blocks(case["K"])):
        k = slice(BLOCK * j, BLOCK * (j + 1))
        columns = t["b_scale"][:, j].double().repeat_interleave(BLOCK)[:case["N"]]
        out += (a[:, k] @ b[:, k].T.contiguous()) * t["a_scale"][:, j].double()[:, None] * columns
    return {"out": out}


def _exact_rotate(case, t):
    """Row by row of the requests; each pair of dims as a complex number."""
    R = case["R"]
    starts, lengths = t["starts"].tolist(), t["lengths"].tolist()
    offsets = t["offsets"].tolist() if "offsets" in t else [0] * len(lengths)
    pos = [offsets[b] + lengths[b] - (starts[b + 1] - r) for b in range(len(lengths)) for r in range(starts[b], starts[b + 1])]
    at = torch.tensor(pos, dtype=torch.long, device=t["cos"].device)
    turn = torch.complex(t["cos"][at].double(), t["sin"][at].double())[:, None]
    out = {}
    for x in ("q", "k"):
        y = t[x][:len(pos)].double()
        if x + "_weight" in t:
            y = y / torch.sqrt((y * y).sum(-1, keepdim=True) / case["D"] + 1e-6) * t[x + "_weight"].double()
        z = torch.zeros(t[x].shape, dtype=torch.float64, device=y.device)
        z[:len(pos), :, R:] = y[..., R:]
        pairs = torch.complex(y[..., 0:R:2], y[..., 1:R:2]) if case["interleaved"] else torch.complex(y[..., :R // 2], y[..., R // 2:R])
        pairs = pairs * turn
        z[:len(pos), :, :R] = torch.stack([pairs.real, pairs.imag], -1).flatten(-2) if case["interleaved"] else torch.cat([pairs.real, pairs.imag], -1)
        out[x + "_out"] = z
    return out


def _exact_prefix(case, t):
    hkv, G, D, page = (case[k] for k in ("hkv", "G", "D", "page"))
    starts, lengths, members, prefix = (t[k].tolist() for k in ("starts", "lengths", "members", "prefix_lengths"))
    out = torch.zeros(t["out"].shape, dtype=torch.float64, device=t["out"].device)

    def held(x, pages, n, h):
        pages = pages[:-(-n // page)].long()
        return (t[x + "_cache"][pages, h].double() * t[x + "_scale"][pages, h].double()[:, None, None]).reshape(-1, D)[:n]

    for h in range(hkv):
        shared = [(held("k", t["prefix_table"][g], n, h), held("v", t["prefix_table"][g], n, h)) for g, n in enumerate(prefix)]
        for b, total in enumerate(lengths):
            n = starts[b + 1] - starts[b]
            if not n:
                continue
            keys, values = held("k", t["page_table"][b], total, h), held("v", t["page_table"][b], total, h)
            ahead = 0
            for g in range(len(prefix)):
                if members[g] <= b < members[g + 1]:
                    keys, values, ahead = torch.cat([shared[g][0], keys]), torch.cat([shared[g][1], values]), prefix[g]
            at = torch.arange(len(keys), device=keys.device)
            q = t["q"][starts[b]:starts[b] + n, h * G:(h + 1) * G].double()
            s = (q.reshape(-1, D) @ keys.T.contiguous() / math.sqrt(D)).reshape(n, G, -1)
            last = (ahead + total - n + torch.arange(n, device=keys.device))[:, None, None]
            s = s.masked_fill(at > last, -math.inf)
            out[starts[b]:starts[b] + n, h * G:(h + 1) * G] = (torch.softmax(s, -1).reshape(-1, len(keys)) @ values).reshape(n, G, D)
    return {"out": out}


def exact(case, seed):
    t, _ = _inputs(case, seed)
    return {"quantize": _exact_quantize, "matmul": _exact_matmul, "rotate": _exact_rotate, "prefix": _exact_prefix}[case["kind"]](case, t)
