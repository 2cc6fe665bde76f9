"""One layer's keys and values of many requests, in pages of 8-bit codes with a scale for each page and head
(include/rai_hip.h, "many requests over a paged 8-bit cache").  A step:

    plan = ops.kv_plan(lens, add, free_pages, taken, tables, page, rows)         # once for all layers
    q, k = ops.rope_positions(q, plan.positions, freqs), ops.rope_positions(k, plan.positions, freqs)
    cache.append(k, v, plan.runs)
    out = cache.attention(q, tables, plan.starts, plan.lens, scale)
"""
from __future__ import annotations

from ._lib import KV_FORMAT, U8, F32, call
from .hip import HipTensor
from .ops import _d, full


class KvCache:
    def __init__(self, pages, kv_heads, head_dim, page, format="e4m3", dev=0):
        f = (head_dim + 15) // 16 * 16
        self.page, self.format, self.dev = int(page), format, dev
        self.k = full(0, (pages, kv_heads, page, f), U8, dev)
        self.v = full(0, (pages, kv_heads, f, page), U8, dev)
        self.k_scale = full(0, (pages, kv_heads), F32, dev)
        self.v_scale = full(0, (pages, kv_heads), F32, dev)

    def _parts(self):
        return KV_FORMAT[self.format], _d(self.k), _d(self.v), _d(self.k_scale), _d(self.v_scale)

    def append(self, k, v, runs):
        """rai_hip_kv_append: k and v [rows, kv heads, head_dim] to where `runs` says."""
        call("rai_hip_kv_append", self.dev, _d(k), _d(v), _d(runs), *self._parts())

    def attention(self, q, tables, starts, lens, scale, window=0, out=None):
        """rai_hip_kv_attention: q [rows, heads, head_dim] -> the same shape.  `out` (optional) keeps its rows that belong to no request."""
        out = HipTensor.empty(q.shape, q.dtype, q.dev) if out is None else out
        call("rai_hip_kv_attention", self.dev, _d(q), _d(tables), _d(starts), _d(lens), *self._parts(), float(scale), int(window), _d(out))
        return out
