"""Batches over the paged cache (kv_models.py) in which every key shows in the result: scores near to each other, so that no few keys hold the whole softmax, and values
that give each key, or each sixteen keys, a feature to themselves."""
import numpy as np

from oracle import kv_cache as O
from tests.kv_models import HALF_STEP, Batch


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
