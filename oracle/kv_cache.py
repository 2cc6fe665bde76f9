"""Serving many requests over a paged 8-bit cache, restated in NumPy with 64-bit arithmetic: test infrastructure.  It has no counterpart
in the reference; the definitions are those of include/rai_hip.h."""
import math

import numpy as np

LARGEST = {"e4m3": 448.0, "int8": 127.0}
MOST_EXP = {"e4m3": 119, "int8": 121}
# code -> value of e4m3: sign, 4 bits of exponent (bias 7), 3 of mantissa, the last code of each sign no number
_E4M3 = np.array([(m / 8 * 2.0 ** -6 if e == 0 else (1 + m / 8) * 2.0 ** (e - 7)) for e in range(16) for m in range(8)])
_E4M3[127] = np.nan


def values(codes, form):
    codes = np.asarray(codes, dtype=np.uint8)
    if form == "int8":
        return codes.view(np.int8).astype(np.float64)
    return np.where(codes < 128, _E4M3[codes & 127], -_E4M3[codes & 127])


def codes(x, form):
    """Nearest code, the even one of two as near; NaN is zero, what lies outside the largest."""
    x = np.nan_to_num(np.asarray(x, dtype=np.float64), nan=0.0, posinf=np.inf, neginf=-np.inf)
    x = np.clip(x, -LARGEST[form], LARGEST[form])
    if form == "int8":
        return np.rint(x).astype(np.int8).view(np.uint8)
    grid, mag = _E4M3[:127], np.abs(x)
    hi = np.clip(np.searchsorted(grid, mag), 1, 126)
    below, above = mag - grid[hi - 1], grid[hi] - mag
    c = np.where((below > above) | ((below == above) & (hi % 2 == 0)), hi, hi - 1)
    return (c + 128 * np.signbit(x)).astype(np.uint8)


def scale_of(largest, form):
    """2^e, e the least whole number with largest <= LARGEST 2^e, within what is allowed."""
    if not largest > 0:
        return 2.0 ** -100
    e = math.frexp(largest / LARGEST[form])
    e = e[1] - 1 if e[0] == 0.5 else e[1]
    return 2.0 ** min(max(e, -100), MOST_EXP[form])


def plan(lens, add, free, taken, tables, page, n_rows, n_runs):
    """-> (tables, lens, taken, starts, positions, runs, refused)"""
    R, M = tables.shape
    tables, out_lens = tables.copy(), np.array(lens, dtype=np.int64)
    starts, positions, runs = np.zeros(R + 1, np.int64), np.full(n_rows, -1, np.int64), []
    refused, asked, given = 0, 0, 0
    room = len(free) - taken if 0 <= taken <= len(free) else 0
    for r in range(R):
        n, a = int(lens[r]), int(add[r])
        starts[r + 1] = starts[r] + max(a, 0)
        ok = n >= 0 and a >= 0 and n + a <= M * page and starts[r + 1] <= n_rows
        held = -(-n // page)
        need = -(-(n + a) // page) - held if ok else 0
        asked += need
        if not ok or (need and asked > room):
            refused += 1
            continue
        for j in range(need):
            tables[r, held + j] = free[taken + asked - need + j]
            given = asked
        out_lens[r] = n + a
        positions[starts[r]:starts[r + 1]] = n + np.arange(a)
        p = n
        while p < n + a:
            count = min(n + a, (p // page + 1) * page) - p
            runs.append((tables[r, p // page], p % page, starts[r] + p - n, count))
            p += count
    runs += [(0, 0, 0, 0)] * (n_runs - len(runs))
    return tables, out_lens, taken + given, starts, positions, np.array(runs, np.uint32).reshape(n_runs, 4).T, refused


def frequencies(rot, base, factor=0.0, low=1.0, high=4.0, original=8192.0):
    f = float(base) ** (-2.0 * np.arange(rot // 2) / rot)
    if factor > 0:
        s = np.clip((original * f / (2 * math.pi) - low) / (high - low), 0, 1)
        f = (1 - s) * f / factor + s * f
    return f


def rope(x, positions, freqs, interleaved, inverse, magnitude):
    x, half = np.asarray(x, dtype=np.float64), len(freqs)
    i = np.arange(half)
    a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + half)
    angle = np.asarray(positions, dtype=np.float64)[:, None, None] * freqs * (-1 if inverse else 1)
    out = x.copy()
    out[..., a] = magnitude * (x[..., a] * np.cos(angle) - x[..., b] * np.sin(angle))
    out[..., b] = magnitude * (x[..., b] * np.cos(angle) + x[..., a] * np.sin(angle))
    return out


def append(new, runs, form, cache, scales, transposed):
    """One side (keys, or values: transposed) of an append, in copies; -> (cache, scales, refused)"""
    cache, scales = cache.copy(), scales.astype(np.float64)
    new = np.asarray(new, dtype=np.float64)
    pages, page, f = cache.shape[0], cache.shape[3 if transposed else 2], cache.shape[2 if transposed else 3]
    seen, refused = set(), 0
    for p, at, row, count in np.asarray(runs, dtype=np.int64).T:
        if count == 0:
            continue
        bad = p in seen or p >= pages or at + count > page or row + count > new.shape[0]
        seen.add(p)
        if bad:
            refused += 1
            continue
        for h in range(new.shape[1]):
            held = cache[p, h].T if transposed else cache[p, h]     # [slot, feature], a view
            x = new[row:row + count, h]
            finite = np.abs(x[np.isfinite(x)])
            s = scale_of(finite.max() if finite.size else 0.0, form)
            if at > 0:
                s = max(s, scales[p, h])
                held[:at] = codes(values(held[:at], form) * (scales[p, h] / s), form)
            held[at:at + count] = 0
            held[at:at + count, :x.shape[1]] = codes(x / s, form)
            scales[p, h] = s
    return cache, scales.astype(np.float32), refused


def attention(q, tables, starts, lens, form, k, v, k_scale, v_scale, page, scale, window=0):
    """-> (out, spread): the sums in 64 bits, and sum p |v| with the same weights, which errors of the weights are measured against,
    and how far rounding 24-bit scores can move a weight, relative, as the largest of a row."""
    q = np.asarray(q, dtype=np.float64)
    N, Hq, D = q.shape
    kd = values(k, form)[..., :D] * np.asarray(k_scale, np.float64)[:, :, None, None]
    vd = values(v, form)[:, :, :D] * np.asarray(v_scale, np.float64)[:, :, None, None]
    out, spread, slip = np.zeros((N, Hq, D)), np.zeros((N, Hq, D)), np.zeros((N, Hq, 1))
    G = Hq // k.shape[1]
    for r in range(len(lens)):
        lo, hi = (min(max(int(x), 0), N) for x in starts[r:r + 2])      # of its rows those that are there
        length = min(max(int(lens[r]), 0), tables.shape[1] * page)      # of its tokens those that its table holds
        if hi <= lo or length == 0:
            continue
        ids = [int(t) for t in tables[r, :-(-length // page)]]
        there = np.repeat([t < k.shape[0] for t in ids], page)[:length]
        ids = [t if t < k.shape[0] else 0 for t in ids]
        p = int(lens[r]) - int(starts[r + 1]) + np.arange(lo, hi)[:, None]
        j = np.arange(length)[None]
        hidden = (j > p) | ~there
        if window:
            hidden |= j <= p - window
        for h in range(Hq):
            kk = kd[ids, h // G].reshape(-1, D)[:length]
            vv = np.where(there[:, None], vd[ids, h // G].transpose(0, 2, 1).reshape(-1, D)[:length], 0.0)
            kk = np.where(there[:, None], kk, 0.0)
            x = q[lo:hi, h]
            s = np.where(hidden, -np.inf, x @ kk.T * scale)
            top = np.max(s, 1, keepdims=True)
            w = np.where(hidden, 0.0, np.exp(s - np.where(np.isfinite(top), top, 0.0)))
            total = w.sum(1, keepdims=True)
            w = np.divide(w, total, out=np.zeros_like(w), where=total > 0)
            out[lo:hi, h] = w @ vv
            spread[lo:hi, h] = w @ np.abs(vv)
            size = np.where(hidden, 0.0, np.abs(x) @ np.abs(kk).T * abs(scale))
            slip[lo:hi, h] = size.max(1, keepdims=True)
    return out, spread, slip
