"""Batches over the paged cache (kv_models.py) in which every key shows in the result: scores near to each other, so that no few keys hold the whole softmax, and values
that give each key, or each sixteen keys, a feature to themselves."""
import numpy as np

from oracle import kv_cache as O
from tests.kv_models import HALF_STEP, Batch, rows


class Seen(Batch):
    """Keys of size one.  Key j's value is one at feature (j // width + 7 head) % dim, in pages whose scales are 1/2, 1 or 2, and zero elsewhere."""

    def __init__(self, rng, total, new, page, kv_heads, dim, form, width, **kw):
        super().__init__(rng, total, new, page, kv_heads, dim, form, **kw)
        codes = O.codes(np.clip(rng.standard_normal((self.pages, kv_heads, page, self.F)) * 32, -120, 120), form)
        one = int(O.codes([1.0], form)[0])
        h = np.arange(kv_heads)
        for r, t in enumerate(self.total):
            for i in range(-(-t // page)):
                p, n = self.tables[r, i], min(page, t - i * page)
                self.k[p, :, :n] = codes[p, :, :n]
                self.k[p, :, :n, dim:] = 0
                self.k_scale[p] = 1 / 32
                self.v[p, :, :, :n] = 0
                for s in range(n):
                    self.v[p, h, ((i * page + s) // width + 7 * h) % dim, s] = one
                self.v_scale[p] = 2.0 ** rng.integers(-1, 2, kv_heads)


def tight_bound(want, spread, slip, dt, dim, keys):
    """As kv_models.attention_bound, with the weights of 16-bit rows rounded to 16 significant bits (2^-16) and those of f32 rows to 24: scores (dim + 4) 2^-24 of sum
    |q k| scale and that again for the row's largest, exp2 2^-22, sums over the keys and their total (keys + 64) 2^-24 each, the output rounded to its type."""
    weight = 2.0 ** -24 if dt == "f32" else 2.0 ** -16
    relative = weight + 2 * (dim + 4) * 2.0 ** -24 * slip + 2.0 ** -21 + 2 * (keys + 64) * 2.0 ** -24
    return spread * relative + np.abs(want) * HALF_STEP[dt] * 1.01 + (2.0 ** -25 if dt == "f16" else 0.0)


def want(b, q, dt, scale, window=0):
    """-> (the sums in 64 bits, how far a kernel may be off)"""
    out, spread, slip = O.attention(q, b.tables, b.starts, b.lens, b.form, b.k, b.v, b.k_scale, b.v_scale, b.page, scale, window)
    return out, tight_bound(out, spread, slip, dt, b.dim, max(b.total))


# total, new, page, key heads, heads, features, window, form, pages of a table (None: what the longest needs).  Whole tiles and tiles that workers share, of few columns, of many,
# and both; parts of a tile over few workers and over hundreds; tables far wider than any context.
CASES = {
    "one row, a head": ([9000], [1], 16, 1, 8, 256, 0, "e4m3", None),
    "three rows": ([5000, 3100, 4777], [1, 1, 1], 16, 2, 12, 128, 0, "e4m3", None),
    "five rows of one": ([4000], [5], 16, 2, 12, 80, 0, "int8", None),
    "two chunks": ([3000, 2100], [150, 97], 16, 2, 4, 64, 0, "e4m3", None),
    "many requests": ([300 - 3 * i for i in range(70)], [1] * 70, 16, 8, 8, 80, 0, "e4m3", None),
    "whole tiles of few": ([1200, 900, 64, 777], [1, 1, 1, 1], 32, 8, 32, 128, 0, "int8", None),
    "few and many": ([6000, 3000, 700, 5000, 1, 0], [1, 130, 1, 65, 1, 0], 16, 2, 12, 128, 0, "e4m3", None),
    "few and many, one key head": ([2500, 4100, 4100], [200, 1, 2], 128, 1, 6, 256, 0, "int8", None),
    "few and many in a window": ([2500, 4100, 3000], [200, 1, 2], 128, 2, 12, 128, 1900, "e4m3", None),
    "many, shared": ([1500, 90, 257, 40], [150, 60, 57, 1], 32, 2, 40, 128, 0, "int8", None),
    "many, whole": ([900, 300], [200, 120], 64, 1, 40, 64, 0, "e4m3", None),
    "many in a window": ([1400, 600], [250, 200], 64, 1, 41, 64, 700, "e4m3", None),
    "few workers to a head": ([5000, 2900, 170], [1, 30, 1], 64, 20, 20, 80, 0, "int8", None),
    "a wide table": ([777], [1], 16, 2, 12, 128, 0, "e4m3", 512),
    "a wider table": ([777], [1], 16, 2, 12, 128, 0, "int8", 8192),
    "chunks under a wide table": ([500, 300], [24, 3], 64, 2, 12, 128, 0, "e4m3", 2048),
}


def case(name, dt):
    total, new, page, kv, heads, dim, window, form, table = CASES[name]
    rng = np.random.default_rng(sum(total) + dim)
    b = Seen(rng, total, new, page, kv, dim, form, 16, table=table)
    return b, heads, window, 0.5 * dim ** -0.5, rows(rng, (b.N, heads, dim), dt)


def least_seen(b, q, dt, heads, window, scale, step=64):
    """Of the last row of every request and of three heads: by how many times the bound the result moves if one step of 64 keys is left out, or counted twice; the least."""
    least, G = np.inf, heads // b.k.shape[1]
    for r in range(len(b.total)):
        t = b.total[r]
        if b.new[r] == 0:
            continue
        ids = b.tables[r, :-(-t // b.page)]
        first = max(0, t - window) if window else 0
        for h in {0, heads // 2, heads - 1}:
            k = (O.values(b.k[ids, h // G], b.form) * b.k_scale[ids, h // G, None, None]).reshape(-1, b.F)[first:t, :b.dim]
            v = (O.values(b.v[ids, h // G], b.form) * b.v_scale[ids, h // G, None, None]).transpose(0, 2, 1).reshape(-1, b.F)[first:t, :b.dim]
            x = q[b.starts[r + 1] - 1, h].astype(np.float64)
            s = k @ x * scale
            w = np.exp(s - s.max())
            edges = np.unique([0] + [e - first for e in range(step, t, step) if e > first])
            sums, totals = np.add.reduceat(w[:, None] * v, edges, 0), np.add.reduceat(w, edges)
            out = sums.sum(0) / totals.sum()
            bound = tight_bound(out, out, np.max(np.abs(k) @ np.abs(x)) * scale, dt, b.dim, max(b.total))
            if len(edges) == 1:
                continue   # a row's only step
            for sign in (-1, 1):
                moved = (sums.sum(0) + sign * sums) / (totals.sum() + sign * totals)[:, None]
                least = min(least, np.max(np.abs(moved - out) / np.maximum(bound, 1e-300), 1).min())
    return least
