"""Plain forms of the paged operators in 64 bits (numpy), shared by their tests."""

import numpy as np

TOP = {"i8": 127.0, "e4m3": 448.0}


def _e4m3_values():
    """Value of each code 0 .. 126 (sign apart); 127 is NaN."""
    c = np.arange(127)
    e, m = c >> 3, c & 7
    return np.where(e == 0, m * 2.0 ** -9, (8 + m) * 2.0 ** (e - 10.0))


E4M3 = _e4m3_values()


def decode(codes, kind):
    """Codes (int8, or uint8 bits of e4m3) as float64."""
    if kind == "i8":
        return codes.astype(np.float64)
    bits = codes.astype(np.int64) & 0xFF
    mag = np.where((bits & 0x7F) == 0x7F, np.nan, E4M3[np.minimum(bits & 0x7F, 126)])
    return np.where(bits & 0x80, -mag, mag)


def encode(y, kind):
    """The nearest code of each float64 (ties to even), saturating; NaN: the e4m3 NaN, or 0."""
    nan = np.isnan(y)
    y = np.where(nan, 0.0, np.clip(y, -TOP[kind], TOP[kind]))
    if kind == "i8":
        return np.rint(y).astype(np.int8)
    mag = np.abs(y)
    hi = np.clip(np.searchsorted(E4M3, mag), 1, 126)
    lo = hi - 1
    down, up = mag - E4M3[lo], E4M3[hi] - mag
    code = np.where((up < down) | ((up == down) & (hi % 2 == 0)), hi, lo)
    return np.where(nan, 0x7F, code | np.where(np.signbit(y), 0x80, 0)).astype(np.uint8)


def f32(x):
    """The nearest float32 value, in 64 bits."""
    with np.errstate(over="ignore"):
        return np.asarray(x, np.float64).astype(np.float32).astype(np.float64)


def plan(lengths, counts, table, free, used, page, rows):
    table, slots = table.copy(), np.full(rows, -1, np.int64)
    starts = np.concatenate([[0], np.cumsum(counts)])
    for b, (n, c) in enumerate(zip(lengths, counts)):
        for j in range(-(-n // page), -(-(n + c) // page)):
            table[b, j] = free[used]
            used += 1
        for i in range(c):
            slots[starts[b] + i] = table[b, (n + i) // page] * page + (n + i) % page
    return {"page_table": table, "slots": slots, "starts": starts, "new_lengths": lengths + counts, "new_used": np.array([used])}


def runs(slots, page):
    """Runs of neighbouring rows of one page: (page, rows)."""
    out, last = [], None
    for r, s in enumerate(slots):
        p = int(s) // page if s >= 0 else None
        if p is not None and p == last:
            out[-1][1].append(r)
        elif p is not None:
            out.append((p, [r]))
        last = p
    return out


def store(x, slots, codes, scale, kind):
    """x [T, H, D] float64, codes [P, H, page, D], scale [P, H] float32: new codes and scales."""
    codes, scale, page = codes.copy(), scale.copy(), codes.shape[2]
    for p, rows in runs(slots, page):
        off = [int(slots[r]) - p * page for r in rows]
        low, new = min(off), x[rows]
        finite = np.where(np.isfinite(new), np.abs(new), 0.0)
        s = np.maximum(f32(finite.max((0, 2)) / TOP[kind]), 2.0 ** -126)
        old = scale[p].astype(np.float64)
        if low:
            s = np.maximum(s, old)
        inv = f32(1.0 / s)
        if low:
            kept = encode(f32(f32(decode(codes[p, :, :low], kind) * old[:, None, None]) * inv[:, None, None]), kind)
            codes[p, :, :low] = np.where((s > old)[:, None, None], kept, codes[p, :, :low])
        for r, o in zip(rows, off):
            with np.errstate(invalid="ignore"):
                codes[p, :, o] = encode(f32(x[r] * inv[:, None]), kind)
        scale[p] = s
    return codes, scale


def attend(q, k, v, k_scale, v_scale, table, lengths, starts, scale, window=0):
    """q [T, HQ, D], k, v [P, H, page, D] as numbers, all float64: out, lse, and what bounds an evaluation's
    error: sum(w |v|), the largest sum(|q k|) scale, sum(|v|)."""
    T, HQ, D = q.shape
    P, H, page, _ = k.shape
    G = HQ // H
    out, lse = np.full((T, HQ, D), np.nan), np.full((T, HQ), np.nan)
    spread, swing, bulk = np.zeros((T, HQ, D)), np.zeros((T, HQ)), np.zeros((T, HQ, D))
    for b in range(len(lengths)):
        n, L = starts[b + 1] - starts[b], int(lengths[b])
        pages = table[b, :-(-L // page)]
        kk = (k[pages] * k_scale[pages][:, :, None, None]).transpose(1, 0, 2, 3).reshape(H, -1, D)[:, :L]
        vv = (v[pages] * v_scale[pages][:, :, None, None]).transpose(1, 0, 2, 3).reshape(H, -1, D)[:, :L]
        for i in range(n):
            pos, r = L - n + i, starts[b] + i
            lo = max(0, pos + 1 - window) if window else 0
            if pos < 0 or pos + 1 <= lo:
                out[r], lse[r] = 0.0, -np.inf
                continue
            for h in range(HQ):
                kt, vt = kk[h // G, lo:pos + 1], vv[h // G, lo:pos + 1]
                s = kt @ q[r, h] * scale
                m = s.max()
                e = np.exp(s - m)
                out[r, h] = e @ vt / e.sum()
                lse[r, h] = m + np.log(e.sum())
                spread[r, h] = e @ np.abs(vt) / e.sum()
                bulk[r, h] = np.abs(vt).sum(0)
                swing[r, h] = (np.abs(kt) @ np.abs(q[r, h])).max() * abs(scale)
    return out, lse, spread, swing, bulk
