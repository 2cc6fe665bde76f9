"""Requests over a paged cache, as the tests of rai_hip_kv_* make them: lengths, tables with pages in any order, codes and scales."""
import numpy as np

from oracle import kv_cache as O
from oracle.dtypes import rnd
from rai_amd.hip import HipTensor

HALF_STEP = {"bf16": 2.0 ** -8, "f16": 2.0 ** -11, "f32": 2.0 ** -24}   # torch.finfo(t).eps / 2


def dev(a, dt):
    return HipTensor.from_storage(np.ascontiguousarray(a), dt)


class Batch:
    """Requests of `total` tokens, the last `new` of each being this step's, their tables over a pool of pages in a shuffled order."""

    def __init__(self, rng, total, new, page, kv_heads, dim, form, spare=2, table=None, garbage=True):
        self.total, self.new, self.page, self.dim, self.form = list(total), list(new), page, dim, form
        self.F = (dim + 15) // 16 * 16
        used = [-(-t // page) for t in total]
        self.pages = sum(used) + spare
        self.M = max(used + [1]) if table is None else table
        order, at = rng.permutation(self.pages), 0
        self.tables = rng.integers(0, 2 ** 32, (len(total), self.M), dtype=np.uint32)   # entries behind a request's pages are anything
        for r, n in enumerate(used):
            self.tables[r, :n] = order[at:at + n]
            at += n
        self.starts = np.concatenate([[0], np.cumsum(new)]).astype(np.int64)
        self.lens = np.array(total, dtype=np.int64)
        self.N = int(self.starts[-1])
        shape = (self.pages, kv_heads, page, self.F)
        x = rng.standard_normal(shape) * 10.0 ** rng.uniform(-1, 1, (self.pages, kv_heads, 1, 1))
        y = rng.standard_normal(shape) * 10.0 ** rng.uniform(-1, 1, (self.pages, kv_heads, 1, 1))
        x[..., dim:] = y[..., dim:] = 0
        self.k_scale, self.v_scale = (np.vectorize(lambda m: O.scale_of(m, form))(np.abs(t).max((2, 3))).astype(np.float32) for t in (x, y))
        self.k = O.codes(x / self.k_scale[:, :, None, None], form)
        self.v = np.ascontiguousarray(O.codes(y / self.v_scale[:, :, None, None], form).transpose(0, 1, 3, 2))
        if garbage:   # slots no request has written: NaN where the format has one
            mark = 0x7f if form == "e4m3" else 0x80
            written = np.zeros((self.pages, page), bool)
            for r, t in enumerate(total):
                for i in range(used[r]):
                    written[self.tables[r, i], :min(page, t - i * page)] = True
            for p in range(self.pages):
                self.k[p][:, ~written[p]] = mark
                self.v[p][:, :, ~written[p]] = mark
                if not written[p].any():
                    self.k_scale[p] = self.v_scale[p] = np.nan

    def cache(self):
        from rai_amd.kv_cache import KvCache

        c = KvCache.__new__(KvCache)
        c.page, c.format, c.dev = self.page, self.form, 0
        c.k, c.v, c.k_scale, c.v_scale = dev(self.k, "u8"), dev(self.v, "u8"), dev(self.k_scale, "f32"), dev(self.v_scale, "f32")
        return c


def attention_bound(want, spread, slip, dt, dim, keys):
    """How far a correct kernel may be off, per element.  A weight in f32 carries the scores' rounding (dim products and their sum, the scale: at
    most (dim + 4) 2^-24 of sum |q k| scale, and that again for the row's largest, exp2 itself 2^-22) and is rounded once more for the
    second product (bf16: 2^-8; f16: two bf16, 2^-16; f32: three, 2^-24); sums over the keys in f32 add at most (keys + 64) 2^-24, as
    does their total; the output is rounded to its type."""
    weight = {"bf16": 2.0 ** -8, "f16": 2.0 ** -16, "f32": 2.0 ** -24}[dt]
    relative = weight + 2 * (dim + 4) * 2.0 ** -24 * slip + 2.0 ** -21 + 2 * (keys + 64) * 2.0 ** -24
    tiny = 2.0 ** -25 if dt == "f16" else 0.0   # half the least f16
    return spread * relative + np.abs(want) * HALF_STEP[dt] * 1.01 + tiny


def rows(rng, shape, dt, scale=1.0):
    return rnd((rng.standard_normal(shape) * scale).astype(np.float32), dt)
