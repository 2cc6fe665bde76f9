"""Serving many requests over a paged 8-bit cache: each operator against 64 bits, and a run of them together."""
import threading

import numpy as np
import pytest

from oracle import kv_cache as O
from oracle.dtypes import rnd
from rai_amd import ops
from rai_amd._lib import call
from rai_amd.hip import HipTensor
from tests.kv_models import HALF_STEP, Batch, attention_bound, dev, rows
from tests.util import down, up

pytestmark = pytest.mark.gpu


def same(got, want, what):
    assert np.array_equal(got, want, equal_nan=got.dtype.kind == "f"), what


# ------------------------------------------------------------------ plan
def plan_case(rng, R, page, M, most, room=None, extra_rows=0):
    add = rng.integers(0, most + 1, R)
    lens = rng.integers(0, np.maximum(M * page - add, 0) + 1)
    need = int((-(-(lens + add) // page) - -(-lens // page)).sum())
    order = rng.permutation(R * M + need + 16).astype(np.uint32)
    free = order[R * M:R * M + 2 + (need if room is None else room)]
    return lens, add, free, 2, order[:R * M].reshape(R, M), int(add.sum()) + extra_rows


def check_plan(lens, add, free, taken, tables, n, page, in_place=True, extra_runs=0):
    R, M = tables.shape
    w = min(n, n // page + 2 * R) + extra_runs
    want = O.plan(lens, add, free, taken, tables, page, n, w)
    t = dev(tables, "u32")
    out_t = t if in_place else HipTensor.empty((R, M), "u32")
    lens_d, add_d = dev(np.asarray(lens, np.int64), "i64"), dev(np.asarray(add, np.int64), "i64")
    outs = [HipTensor.empty(s, d) for s, d in (((R,), "i64"), ((1,), "i64"), ((R + 1,), "i64"), ((n,), "i64"), ((4, w), "u32"))]
    ops.index_errors()
    for _ in range(2):   # a second call on the same inputs says the same
        args = [lens_d, add_d, dev(free, "u32"), dev(np.array([taken], np.int64), "i64"), t]
        call("rai_hip_kv_plan", 0, *(a.desc() for a in args), page, out_t.desc(), *(o.desc() for o in outs))
        got = [out_t.to_storage()] + [o.to_storage() for o in outs]
        assert ops.index_errors() == want[6]
        for g, wnt, what in zip(got, [want[0], want[1], np.array([want[2]])] + list(want[3:6]), ("tables", "lens", "taken", "starts", "positions", "runs")):
            same(g, wnt, what)


@pytest.mark.parametrize("R,page,M,most", [(1, 16, 1, 1), (1, 16, 4, 64), (3, 16, 8, 40), (64, 16, 12, 1), (257, 32, 5, 30), (700, 64, 3, 190), (1000, 16, 20, 3), (4096, 128, 2, 2), (5, 256, 40, 9000)])
def test_plan(hip, R, page, M, most):
    rng = np.random.default_rng(R * 1000 + page)
    check_plan(*plan_case(rng, R, page, M, min(most, M * page)), page)
    check_plan(*plan_case(rng, R, page, M, min(most, M * page), extra_rows=37), page, in_place=False, extra_runs=5)


@pytest.mark.parametrize("room", [0, 1, 7, 30])
def test_plan_with_too_few_pages(hip, room):
    rng = np.random.default_rng(room)
    check_plan(*plan_case(rng, 90, 16, 12, 50, room=room), 16)


def test_plan_refuses_what_does_not_fit(hip):
    lens, add = [16, -1, 40, 0, 128, 100, 5, 2 ** 62, 3], [16, 4, -7, 0, 1, 28, 2 ** 61, 2 ** 62, 2]
    tables = np.arange(9 * 8, dtype=np.uint32).reshape(9, 8)
    # rows behind the request of 2^61 tokens are past N: everything from there on is refused
    R, n, w = 9, 60, 60
    t = dev(tables, "u32")
    ops.index_errors()
    p = ops.kv_plan(dev(np.array(lens), "i64"), dev(np.array(add), "i64"), dev(np.arange(100, 140, dtype=np.uint32), "u32"), dev(np.zeros(1, np.int64), "i64"), t, 16, n)
    assert p.lens.to_storage().tolist() == [32, -1, 40, 0, 128, 128, 5, 2 ** 62, 3]
    assert p.starts.to_storage().tolist()[:7] == [0, 16, 20, 20, 20, 21, 49]
    assert ops.index_errors() == 6
    got = p.positions.to_storage()
    assert got.tolist() == list(range(16, 32)) + [-1] * 5 + list(range(100, 128)) + [-1] * 11
    t = t.to_storage()
    assert t[0, :3].tolist() == [0, 100, 2] and t[5].tolist() == list(range(40, 47)) + [101]   # (page 6 of request 5 holds 100 .. 111 already)
    assert p.runs.to_storage()[:, :4].T.tolist() == [[100, 0, 0, 16], [46, 4, 21, 12], [101, 0, 33, 16], [0, 0, 0, 0]]


@pytest.mark.parametrize("taken", [-1, 41, 2 ** 40, 40])
def test_plan_with_no_pages_to_take(hip, taken):
    rng = np.random.default_rng(5)
    tables = rng.permutation(40).astype(np.uint32).reshape(5, 8)
    lens, add, free = [16, 17, 0, 31, 5], [1, 1, 0, 2, 11], np.arange(40, dtype=np.uint32)
    check_plan(lens, add, free, taken, tables, 15, 16)


def test_plan_of_nothing(hip):
    p = ops.kv_plan(*(HipTensor.empty((0,), d) for d in ("i64", "i64", "u32")), dev(np.array([3], np.int64), "i64"), HipTensor.empty((0, 4), "u32"), 16, 5)
    assert p.taken.to_storage().tolist() == [3] and p.starts.to_storage().tolist() == [0] and p.positions.to_storage().tolist() == [-1] * 5
    assert p.runs.shape == (4, 0)


# ------------------------------------------------------------------ rotary positions
def check_rope(rng, shape, dt, rot, inter, inverse, magnitude, far, strides=None):
    N, H, D = shape
    x = rows(rng, shape, dt)
    if strides == "packed":      # heads out of the middle of a wider row
        wide = rows(rng, (N, H + 3, D), dt)
        wide[:, 1:1 + H] = x
        xt = up(wide, dt).narrow(1, 1, H)
    elif strides == "odd":       # rows that begin off every boundary
        flat = rows(rng, (N * (H * D + 1) + 1,), dt)
        v = np.lib.stride_tricks.as_strided(flat[1:], shape, tuple(s * flat.itemsize for s in (H * D + 1, D, 1)))
        x = v.copy()
        xt = HipTensor(up(flat, dt).buf, dt, shape, (H * D + 1, D, 1), 1)
    else:
        xt = up(x, dt)
    p = rng.integers(0, far, N)
    p[0] = -1
    f = O.frequencies(rot, 1e4, 8.0 if far > 10 ** 5 else 0.0)
    got = down(ops.rope_positions(xt, dev(p, "i64"), dev(f, "f64"), inter, inverse, magnitude)).astype(np.float64)
    want = O.rope(x, p, f, inter, inverse, magnitude)
    # cosine and sine: the turn in f32 (2^-25 of a half turn, pi of it an error in the angle), sincospi, the magnitude: below 2^-21 together;
    # two products and a sum 2^-23 of theirs; one rounding to the type
    other = np.abs(x) + np.abs(np.where(np.isin(np.arange(D), np.arange(rot)), np.abs(x).max(-1, keepdims=True), 0))
    bound = HALF_STEP[dt] * 1.01 * np.abs(want) + 2.0 ** -20 * magnitude * other + (2.0 ** -25 if dt == "f16" else 0)
    bad = np.abs(got - want) > bound
    assert not bad.any(), (np.abs(got - want)[bad].max(), np.argwhere(bad)[:3])
    same(got[..., rot:], x[..., rot:].astype(np.float64), "features behind the turned ones")


@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("dt", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("shape,rot", [((1, 1, 64), 64), ((7, 3, 80), 32), ((33, 14, 128), 128), ((130, 5, 72), 40), ((5, 2, 11), 6), ((9, 1, 2), 2), ((3, 2, 256), 0), ((2500, 3, 16), 12)])
def test_rope_positions(hip, shape, rot, dt, inter):
    rng = np.random.default_rng(sum(shape) + rot)
    for strides in (None, "packed", "odd"):
        check_rope(rng, shape, dt, rot, inter, False, 1.0, 3000, strides)
    check_rope(rng, shape, dt, rot, inter, True, 1.2079, 10 ** 6)


def test_rope_gradient_against_differences(hip):
    """sum(y g) over x moved by a step: the inverse turn of g, f32."""
    rng = np.random.default_rng(3)
    x, g, p, f = rows(rng, (4, 2, 20), "f32"), rows(rng, (4, 2, 20), "f32"), np.array([0, 5, 999, 12345]), O.frequencies(16, 1e4)
    for inter in (False, True):
        turn = lambda a, inverse=False: down(ops.rope_positions(up(a, "f32"), dev(p, "i64"), dev(f, "f64"), inter, inverse, 1.5)).astype(np.float64)   # noqa: E731
        grad = turn(g, True)
        for at in [(0, 0, 0), (1, 1, 7), (2, 0, 15), (3, 1, 8), (3, 0, 19)]:
            a, b = x.copy(), x.copy()
            a[at] += 0.5
            b[at] -= 0.5
            num = ((turn(a) - turn(b)) * g).sum() / float(a[at] - b[at])
            # each output of the row is off by 2^-20 of the row's largest values
            assert abs(num - grad[at]) <= 2.0 ** -19 * 1.5 * np.abs(x[at[0], at[1]]).max() * np.abs(g[at[0], at[1]]).sum() + 2.0 ** -20 * 4


@pytest.mark.parametrize("rot", [2, 32, 128, 256])
def test_rope_frequencies(hip, rot):
    for args in [(1e4,), (5e5, 8.0, 1.0, 4.0, 8192.0), (1e6, 4.0, 2.0, 32.0, 4096.0)]:
        got, want = ops.rope_frequencies(rot, *args).to_storage(), O.frequencies(rot, *args)
        assert np.allclose(got, want, rtol=1e-13, atol=0)


# ------------------------------------------------------------------ append
def runs_of(batch, extra=0):
    runs = []
    for r, (t, n) in enumerate(zip(batch.total, batch.new)):
        p = t - n
        while p < t:
            c = min(t, (p // batch.page + 1) * batch.page) - p
            runs.append((batch.tables[r, p // batch.page], p % batch.page, batch.starts[r] + p - (t - n), c))
            p += c
    return np.array(runs + [(0, 0, 0, 0)] * extra, np.uint32).reshape(-1, 4).T


def check_append(batch, k, v, dt, runs, kt=None, vt=None):
    c = batch.cache()
    ops.index_errors()
    c.append(kt or up(k, dt), vt or up(v, dt), dev(runs, "u32"))
    refused = 0
    for name, new, transposed in (("k", k, False), ("v", v, True)):
        want, scale, refused = O.append(new, runs, batch.form, getattr(batch, name), getattr(batch, name + "_scale"), transposed)
        same(getattr(c, name + "_scale").to_storage(), scale, name + " scales")
        same(getattr(c, name).to_storage(), want, name)
    assert ops.index_errors() == refused
    return c


@pytest.mark.parametrize("form", ["e4m3", "int8"])
@pytest.mark.parametrize("dt", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("page,heads,dim,total,new", [
    (16, 2, 128, [1], [1]), (16, 2, 128, [16, 17, 40, 31], [1, 1, 1, 1]), (16, 1, 64, [100, 3, 48], [77, 3, 0]), (32, 3, 80, [33, 95], [2, 64]),
    (64, 2, 72, [64, 200], [64, 137]), (128, 2, 256, [130, 1], [129, 1]), (256, 1, 16, [256, 300], [255, 40]), (16, 2, 11, [19, 33], [5, 20]), (16, 33, 32, [20], [9])])
def test_append(hip, page, heads, dim, total, new, dt, form):
    rng = np.random.default_rng(page + heads + dim)
    b = Batch(rng, total, new, page, heads, dim, form)
    k, v = (rows(rng, (b.N, heads, dim), dt, s) for s in (3.0, 0.01))
    k[rng.random(k.shape) < 0.02] *= 100
    check_append(b, rnd(k, dt), v, dt, runs_of(b, extra=3))


def test_append_of_rows_in_a_packed_projection(hip):
    rng = np.random.default_rng(8)
    for width in (2 + 2 + 4, 7):   # whole 16 bytes between rows or not
        b = Batch(rng, [30, 5, 64], [17, 5, 33], 16, 2, 60, "e4m3")
        wide = rows(rng, (b.N, width, 60), "bf16")
        t = up(wide, "bf16")
        check_append(b, wide[:, 1:3], wide[:, 4:6], "bf16", runs_of(b), t.narrow(1, 1, 2), t.narrow(1, 4, 2))


@pytest.mark.parametrize("form", ["e4m3", "int8"])
def test_append_of_values_that_are_no_numbers(hip, form):
    rng = np.random.default_rng(9)
    b = Batch(rng, [40, 16], [24, 3], 16, 2, 64, form)
    k = rows(rng, (b.N, 2, 64), "f32")
    k[3, 0, :3], k[5, 1] = (np.inf, -np.inf, np.nan), np.nan
    k[20:24, 1] = 0.0
    v = k[::-1].copy()
    v[0] = np.finfo(np.float32).max
    v[1] = 1e-42
    check_append(b, k, v, "f32", runs_of(b))


@pytest.mark.parametrize("form", ["e4m3", "int8"])
def test_append_token_by_token(hip, form):
    """A page filled one token at a time, magnitudes rising and falling: its scale never falls, its codes follow."""
    rng = np.random.default_rng(10)
    b = Batch(rng, [16], [16], 16, 2, 32, form, spare=0)
    for i, m in enumerate([1.0, 0.1, 300.0, 5.0, 5.0, 1e-3, 4000.0, 0.0, 1e5] + [1.0] * 7):
        k, v = (rows(rng, (1, 2, 32), "bf16", m) for _ in range(2))
        runs = np.array([[b.tables[0, 0]], [i], [0], [1]], np.uint32)
        c = check_append(b, k, v, "bf16", runs)
        b.k, b.v, b.k_scale, b.v_scale = (t.to_storage() for t in (c.k, c.v, c.k_scale, c.v_scale))


def test_append_refuses_runs_that_are_not_there(hip):
    rng = np.random.default_rng(11)
    b = Batch(rng, [64, 64], [20, 20], 16, 2, 64, "int8")
    k, v = (rows(rng, (40, 2, 64), "bf16") for _ in range(2))
    p = [int(x) for x in b.tables[0, :4]] + [int(b.tables[1, 0])]
    runs = np.array([(p[0], 3, 0, 5), (b.pages, 0, 0, 1), (2 ** 32 - 1, 0, 0, 1), (p[1], 16, 0, 1), (p[2], 15, 0, 2), (p[3], 0, 39, 2), (p[0], 8, 5, 8), (p[4], 0, 2 ** 32 - 1, 1),
                     (p[1], 0, 0, 16), (0, 0, 0, 0)], np.uint32).T
    check_append(b, k, v, "bf16", runs)


# ------------------------------------------------------------------ attention
def check_attention(batch, q, dt, heads, window=0, scale=None, qt=None, table_cols=0):
    D = batch.dim
    scale = D ** -0.5 if scale is None else scale
    c = batch.cache()
    tables = dev(np.pad(batch.tables, ((0, 0), (0, table_cols)), constant_values=2 ** 32 - 1), "u32")
    got = down(c.attention(qt or up(q, dt), tables, dev(batch.starts, "i64"), dev(batch.lens, "i64"), scale, window)).astype(np.float64)
    want, spread, slip = O.attention(q, batch.tables, batch.starts, batch.lens, batch.form, batch.k, batch.v, batch.k_scale, batch.v_scale, batch.page, scale, window)
    bound = attention_bound(want, spread, slip, dt, D, max(batch.total))
    assert np.isfinite(got).all()
    over = np.abs(got - want) / np.maximum(bound, 1e-300)
    assert not (np.abs(got - want) > bound).any(), f"{over.max()} of the bound at {np.unravel_index(over.argmax(), over.shape)}"


LENGTHS = [([1], [1]), ([64], [1]), ([65, 16, 1, 200, 63], [1] * 5), ([777], [1]), ([300, 40, 130], [70, 40, 1]), ([5, 0, 9], [5, 0, 0]), ([1500, 64, 2000], [3, 64, 1]), ([129] * 3, [33, 0, 128])]


@pytest.mark.parametrize("form", ["e4m3", "int8"])
@pytest.mark.parametrize("dt", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("total,new", LENGTHS)
def test_attention_lengths(hip, total, new, dt, form):
    rng = np.random.default_rng(sum(total))
    b = Batch(rng, total, new, 16, 2, 128, form)
    check_attention(b, rows(rng, (b.N, 12, 128), dt), dt, 12)


@pytest.mark.parametrize("dt", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("heads,kv", [(1, 1), (8, 8), (8, 1), (6, 2), (40, 2), (7, 7), (33, 1)])
@pytest.mark.parametrize("dim", [16, 64, 72, 80, 100, 128, 192, 256])
def test_attention_heads_and_features(hip, dim, heads, kv, dt):
    rng = np.random.default_rng(dim * 100 + heads)
    for form, page, total, new in (("e4m3", 32, [70, 150], [1, 1]), ("int8", 64, [40, 90], [21, 5])):
        b = Batch(rng, total, new, page, kv, dim, form)
        check_attention(b, rows(rng, (b.N, heads, dim), dt), dt, heads)


@pytest.mark.parametrize("page", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("window", [0, 1, 16, 63, 64, 100, 1000])
def test_attention_windows_and_pages(hip, page, window):
    rng = np.random.default_rng(page + window)
    b = Batch(rng, [400, 33, 257, 64], [1, 33, 100, 2], page, 2, 64, "e4m3")
    check_attention(b, rows(rng, (b.N, 8, 64), "bf16"), "bf16", 8, window)
    b = Batch(rng, [400, 33, 257, 64], [1] * 4, page, 2, 64, "int8")
    check_attention(b, rows(rng, (b.N, 8, 64), "f32"), "f32", 8, window)


@pytest.mark.parametrize("dt", ["bf16", "f32"])
@pytest.mark.parametrize("requests,total,new,heads,kv,dim", [(1, 9000, 1, 8, 1, 256), (3, 5000, 1, 12, 2, 128), (1, 4000, 5, 12, 2, 80), (2, 3000, 150, 4, 2, 64), (70, 300, 1, 32, 32, 80)])
def test_attention_of_contexts_over_many_blocks(hip, requests, total, new, heads, kv, dim, dt):
    rng = np.random.default_rng(total)
    lens = [total] + [int(rng.integers(new, total + 1)) for _ in range(requests - 1)]
    b = Batch(rng, lens, [new] * requests, 16, kv, dim, "e4m3")
    check_attention(b, rows(rng, (b.N, heads, dim), dt), dt, heads)


def test_attention_tables_far_longer_than_contexts(hip):
    rng = np.random.default_rng(21)
    b = Batch(rng, [100, 1, 700], [1, 1, 1], 16, 2, 128, "e4m3")
    check_attention(b, rows(rng, (b.N, 4, 128), "bf16"), "bf16", 4, table_cols=5000)


def test_attention_of_sharp_and_flat_scores(hip):
    """Scores that leave one key, scores that are all alike, a scale below zero and one of zero; a maximum that creeps up key by key."""
    rng = np.random.default_rng(22)
    for scale in (20.0, -3.0, 0.0, 1e-4):
        b = Batch(rng, [200, 90], [1, 40], 16, 2, 64, "e4m3")
        check_attention(b, rows(rng, (b.N, 4, 64), "bf16"), "bf16", 4, scale=scale)
    b = Batch(rng, [640], [1], 16, 1, 64, "int8", garbage=False)
    b.k_scale[:] = 1.0
    for i in range(40):
        b.k[b.tables[0, i], 0] = (np.arange(16)[:, None] // 8 + 2 * i).astype(np.int8).view(np.uint8)
    check_attention(b, rnd(np.full((1, 2, 64), 0.05, np.float32), "f32"), "f32", 2, scale=1.0)


@pytest.mark.parametrize("dt", ["bf16", "f32"])
def test_attention_rows_of_a_packed_projection(hip, dt):
    rng = np.random.default_rng(23)
    for H, D, first in ((12, 128, 2), (3, 33, 1)):
        b = Batch(rng, [130, 70], [1, 20], 16, 1 if D == 33 else 2, D, "int8")
        wide = rows(rng, (b.N, H + 5, D), dt)
        check_attention(b, wide[:, first:first + H], dt, H, qt=up(wide, dt).narrow(1, first, H))


def test_attention_leaves_rows_behind_the_last_request(hip):
    rng = np.random.default_rng(24)
    for new in ([1, 1, 1], [1, 40, 3]):
        b = Batch(rng, [1000, 90, 3], new, 16, 2, 64, "e4m3")
        q = up(rows(rng, (b.N + 9, 8, 64), "bf16"), "bf16")
        out = ops.full(7.0, q.shape, "bf16")
        b.cache().attention(q, dev(b.tables, "u32"), dev(b.starts, "i64"), dev(b.lens, "i64"), 0.125, out=out)
        got = down(out)
        assert (got[b.N:] == 7.0).all() and not (got[:b.N] == 7.0).all((1, 2)).any()


def test_attention_rows_that_see_nothing_are_zero(hip):
    """A request whose length was not raised (more rows than tokens), one without tokens, one with a negative length."""
    rng = np.random.default_rng(25)
    for new in ([1, 1, 1, 1], [9, 30, 2, 4]):
        b = Batch(rng, [20, 0, 4, 50], new, 16, 2, 64, "e4m3")
        b.lens[:] = [3, 0, -5, 50]
        c = b.cache()
        q = rows(rng, (b.N, 8, 64), "bf16")
        got = down(c.attention(up(q, "bf16"), dev(b.tables, "u32"), dev(b.starts, "i64"), dev(b.lens, "i64"), 0.125)).astype(np.float64)
        want, spread, slip = O.attention(q, b.tables, b.starts, b.lens, "e4m3", b.k, b.v, b.k_scale, b.v_scale, 16, 0.125)
        assert (np.abs(got - want) <= attention_bound(want, spread, slip, "bf16", 64, 64)).all()
        empty = max(new[0] - 3, 0)
        assert (got[:empty] == 0).all() and (got[b.starts[1]:b.starts[3]] == 0).all() and (got[b.starts[3]:] != 0).any()


def test_attention_hides_pages_that_are_not_there(hip):
    rng = np.random.default_rng(26)
    for new in ([1, 1], [1, 40]):
        b = Batch(rng, [100, 200], new, 16, 1, 64, "int8")
        b.tables[0, 2], b.tables[1, 5], b.tables[1, 6] = b.pages, 2 ** 32 - 1, b.pages + 3
        ops.index_errors()
        check_attention(b, rows(rng, (b.N, 4, 64), "f32"), "f32", 4)
        assert ops.index_errors() > 0
    b = Batch(rng, [100], [1], 16, 1, 64, "int8", table=7)
    q, want = rows(rng, (1, 4, 64), "f32"), None
    b.lens[:] = 112 + 10 ** 12   # past the table: its 112 tokens, of which the last 12 are what memory held
    b.k[b.tables[0, 6]], b.v[b.tables[0, 6]] = 1, 1
    got = down(b.cache().attention(up(q, "f32"), dev(b.tables, "u32"), dev(b.starts, "i64"), dev(b.lens, "i64"), 0.125))
    want = O.attention(q, b.tables, b.starts, np.array([112]), "int8", b.k, b.v, b.k_scale, b.v_scale, 16, 0.125)
    assert (np.abs(got - want[0]) <= attention_bound(*want, "f32", 64, 112)).all() and ops.index_errors() == 1


def test_attention_pages_of_a_shared_prefix(hip):
    rng = np.random.default_rng(27)
    b = Batch(rng, [80, 75, 66], [1, 1, 1], 16, 2, 64, "e4m3")
    b.tables[1:, :4] = b.tables[0, :4]
    check_attention(b, rows(rng, (3, 8, 64), "f16"), "f16", 8)


def test_attention_is_the_same_every_time_and_beside_other_threads(hip):
    """Two threads that call at once: results are those of each alone, bit for bit (they share the device's scratch)."""
    rng = np.random.default_rng(28)
    cases = []
    for total, new, heads, kv, dim, dt in (([5000, 300], [1, 1], 12, 2, 128, "bf16"), ([2000, 900], [30, 1], 4, 4, 64, "f32")):
        b = Batch(rng, total, new, 16, kv, dim, "e4m3")
        cases.append((b.cache(), up(rows(rng, (b.N, heads, dim), dt), dt), dev(b.tables, "u32"), dev(b.starts, "i64"), dev(b.lens, "i64")))
    alone = [c[0].attention(*c[1:], 0.1).to_storage() for c in cases]
    failed = []

    def work(i):
        for _ in range(20):
            if not np.array_equal(cases[i][0].attention(*cases[i][1:], 0.1).to_storage(), alone[i]):
                failed.append(i)

    threads = [threading.Thread(target=work, args=(i,)) for i in (0, 1)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    assert not failed


@pytest.mark.parametrize("dt,heads,kv,dim,window", [("bf16", 12, 2, 128, 0), ("f16", 8, 1, 64, 0), ("f32", 8, 2, 80, 0), ("bf16", 6, 1, 256, 0), ("f32", 4, 1, 256, 700), ("bf16", 12, 2, 128, 1900)])
def test_attention_of_few_and_many_columns_over_long_contexts(hip, dt, heads, kv, dim, window):
    """Both kinds of tiles in one launch, whole ones and ones that workers share, and requests of neither."""
    rng = np.random.default_rng(dim + heads)
    for page, form, total, new in ((16, "e4m3", [6000, 3000, 700, 5000, 1, 0], [1, 200, 1, 65, 1, 0]), (128, "int8", [2500, 4100, 4100], [300, 1, 2])):
        b = Batch(rng, total, new, page, kv, dim, form)
        check_attention(b, rows(rng, (b.N, heads, dim), dt), dt, heads, window)


@pytest.mark.parametrize("longest", [500, 1500])
@pytest.mark.parametrize("dt", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("dim", [16, 64, 72, 80, 100, 128, 192, 256])
def test_attention_of_many_columns(hip, dim, dt, longest):
    """More rows than tiles of few columns hold at once: tiles of many, whole ones and (of long contexts) ones that workers share."""
    rng = np.random.default_rng(dim + longest)
    b = Batch(rng, [longest, 90, 257, 40], [199, 60, 57, 1], 32, 2, dim, "e4m3" if dim % 3 else "int8")
    check_attention(b, rows(rng, (b.N, 40, dim), dt), dt, 40)


@pytest.mark.parametrize("page", [16, 64, 256])
@pytest.mark.parametrize("window", [1, 63, 100, 1000])
def test_attention_of_many_columns_in_windows(hip, page, window):
    rng = np.random.default_rng(page + window)
    for dt, form, heads, kv in (("bf16", "e4m3", 40, 1), ("f32", "int8", 41, 1)):
        b = Batch(rng, [1400, 33, 300, 64], [250, 33, 40, 2], page, kv, 64, form)
        check_attention(b, rows(rng, (b.N, heads, 64), dt), dt, heads, window)


def test_attention_of_many_columns_with_a_scale_below_zero_and_missing_pages(hip):
    rng = np.random.default_rng(35)
    b = Batch(rng, [300, 200], [280, 60], 16, 1, 64, "e4m3")
    q = rows(rng, (b.N, 40, 64), "bf16")
    for scale in (20.0, -3.0, 0.0):
        check_attention(b, q, "bf16", 40, scale=scale)
    b.tables[0, 2], b.tables[1, 5], b.tables[1, 6] = b.pages, 2 ** 32 - 1, b.pages + 3
    ops.index_errors()
    check_attention(b, q, "bf16", 40)
    assert ops.index_errors() > 0


@pytest.mark.parametrize("dt,dim", [("bf16", 64), ("f16", 80), ("f32", 128), ("bf16", 256)])
def test_attention_of_long_contexts_over_many_heads(hip, dt, dim):
    """Few workers to a head, each with parts of a tile or two."""
    rng = np.random.default_rng(dim)
    for new in ([1, 1, 1], [1, 30, 1]):
        b = Batch(rng, [5000, 2900, 170], new, 64, 20, dim, "e4m3")
        check_attention(b, rows(rng, (b.N, 20, dim), dt), dt, 20)


@pytest.mark.parametrize("new", [1, 9])
def test_attention_of_more_requests_than_a_wave_has_lanes(hip, new):
    rng = np.random.default_rng(31 + new)
    total = [int(rng.integers(new, 2600 if i % 40 == 0 else 60)) for i in range(200)]
    b = Batch(rng, total, [new if i % 3 else 0 for i in range(200)], 16, 2, 64, "int8")
    check_attention(b, rows(rng, (b.N, 8, 64), "bf16"), "bf16", 8)


def test_attention_of_tables_that_are_part_of_wider_ones(hip):
    rng = np.random.default_rng(32)
    b = Batch(rng, [700, 90], [1, 40], 16, 2, 64, "e4m3")
    wide = rng.integers(0, 2 ** 32, (2, b.M + 11), dtype=np.uint32)
    wide[:, 3:3 + b.M] = b.tables
    q = rows(rng, (b.N, 8, 64), "bf16")
    got = down(b.cache().attention(up(q, "bf16"), dev(wide, "u32").narrow(1, 3, b.M), dev(b.starts, "i64"), dev(b.lens, "i64"), 0.125)).astype(np.float64)
    want, spread, slip = O.attention(q, b.tables, b.starts, b.lens, b.form, b.k, b.v, b.k_scale, b.v_scale, 16, 0.125)
    assert (np.abs(got - want) <= attention_bound(want, spread, slip, "bf16", 64, 700)).all()


@pytest.mark.parametrize("dt", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("dim", [64, 80, 128, 256])
def test_attention_does_not_see_what_others_left(hip, dim, dt):
    """Registers, LDS, scratch and freed memory full of NaN from the calls before: results are those of a first call, bit for bit."""
    rng = np.random.default_rng(33)
    bad = ops.full(float("nan"), (4, 12, 256, 128), "bf16")
    for total, new in (([70, 150], [1, 1]), ([40, 90], [21, 5]), ([4000, 900], [1, 70])):
        b = Batch(rng, total, new, 32, 1, dim, "e4m3")
        c, q = b.cache(), up(rows(rng, (b.N, 8, dim), dt), dt)
        rest = (dev(b.tables, "u32"), dev(b.starts, "i64"), dev(b.lens, "i64"), dim ** -0.5)
        first = c.attention(q, *rest).to_storage()
        nan = up(np.full((b.N, 8, dim), np.nan, np.float32), dt)
        for _ in range(5):
            ops.attention(bad, bad, bad, 0.1, 1, 0)
            c.attention(nan, *rest)
            held = [ops.full(float("nan"), (n,), "f32") for n in (64, 1024, 16384, 1 << 20)]
            del held
            assert np.array_equal(c.attention(q, *rest).to_storage(), first)


def test_caches_of_more_than_two_to_the_32_bytes(hip):
    """Pages whose codes lie behind 2^32 bytes: rows appended to them, and read back by attention of few columns and of many."""
    from rai_amd.kv_cache import KvCache

    rng = np.random.default_rng(34)
    pages, heads, dim, page = 70000, 2, 256, 128   # 4.6 GB of keys and as much of values
    cache = KvCache(pages, heads, dim, page, "e4m3")
    far = [65537, 69999, 0, 65535, 65536]
    total = [300, 200]
    tables = np.array([far[:3], far[3:] + [1]], np.uint32)
    k, v = (rows(rng, (500, heads, dim), "bf16") for _ in range(2))
    runs = np.array([(far[0], 0, 0, 128), (far[1], 0, 128, 128), (far[2], 0, 256, 44), (far[3], 0, 300, 128), (far[4], 0, 428, 72)], np.uint32).T
    ops.index_errors()
    cache.append(up(k, "bf16"), up(v, "bf16"), dev(runs, "u32"))
    small = [t.narrow(0, 0, 2).to_storage()[[0] * 3 + [1] * 3] * 0 for t in (cache.k, cache.v, cache.k_scale, cache.v_scale)]
    for i, p in enumerate(far):
        for mine, t in zip(small, (cache.k, cache.v, cache.k_scale, cache.v_scale)):
            mine[i] = t.narrow(0, p, 1).to_storage()[0]
    near = np.array([(i, r[1], r[2], r[3]) for i, r in enumerate(runs.T)], np.uint32).T
    for rows_, at, transposed in ((k, 0, False), (v, 1, True)):
        codes, scale, refused = O.append(rows_, near, "e4m3", small[at] * 0, small[2 + at] * 0, transposed)
        same(small[at], codes, "codes")
        same(small[2 + at], scale, "scales")
    table_near = np.array([[0, 1, 2], [3, 4, 5]], np.uint32)
    for new in ([1, 1], [40, 3]):
        starts = np.concatenate([[0], np.cumsum(new)]).astype(np.int64)
        q = rows(rng, (sum(new), 4, dim), "bf16")
        got = down(cache.attention(up(q, "bf16"), dev(tables, "u32"), dev(starts, "i64"), dev(np.array(total, np.int64), "i64"), 0.0625)).astype(np.float64)
        want, spread, slip = O.attention(q, table_near, starts, np.array(total), "e4m3", *small, page, 0.0625)
        assert (np.abs(got - want) <= attention_bound(want, spread, slip, "bf16", dim, 300)).all()
    assert ops.index_errors() == 0


# ------------------------------------------------------------------ together
@pytest.mark.parametrize("form,inter", [("e4m3", False), ("int8", True)])
def test_steps_of_a_serving_loop(hip, form, inter):
    """Requests that come, are fed in portions, decode, pause and end: plan, rope, append and attention of every step against the same in 64
    bits over the codes that the device holds."""
    rng = np.random.default_rng(30)
    Hq, Hkv, D, page, M, R = 6, 2, 80, 16, 8, 4
    from rai_amd.kv_cache import KvCache
    cache = KvCache(R * M, Hkv, D, page, form)
    free = dev(rng.permutation(R * M).astype(np.uint32), "u32")
    taken, tables, lens = dev(np.zeros(1, np.int64), "i64"), ops.full(0, (R, M), "u32"), dev(np.zeros(R, np.int64), "i64")
    freqs = ops.rope_frequencies(32, 1e4)
    f64, total = O.frequencies(32, 1e4), np.zeros(R, np.int64)
    ops.index_errors()
    for add in ([40, 1, 0, 17], [1, 1, 33, 1], [1, 0, 1, 30], [1, 1, 1, 1], [16, 15, 16, 1], [1, 1, 1, 0]):
        add, N = np.array(add, np.int64), sum(add)
        qkv = rows(rng, (N, Hq + 2 * Hkv, D), "bf16")
        t = up(qkv, "bf16")
        plan = ops.kv_plan(lens, dev(add, "i64"), free, taken, tables, page, N)
        turned = ops.rope_positions(t.narrow(1, 0, Hq + Hkv), plan.positions, freqs, inter)
        before = [x.to_storage() for x in (cache.k, cache.v, cache.k_scale, cache.v_scale)]
        cache.append(turned.narrow(1, Hq, Hkv), t.narrow(1, Hq + Hkv, Hkv), plan.runs)
        out = down(cache.attention(turned.narrow(1, 0, Hq), tables, plan.starts, plan.lens, D ** -0.5)).astype(np.float64)
        positions = np.concatenate([n + np.arange(a) for n, a in zip(total, add)])
        total += add
        same(plan.positions.to_storage(), positions, "positions")
        same(plan.lens.to_storage(), total, "lens")
        y = down(turned).astype(np.float64)
        want = O.rope(qkv[:, :Hq + Hkv], positions, f64, inter, False, 1.0)
        assert (np.abs(y - want) <= 2.0 ** -8 * 1.01 * np.abs(want) + 2.0 ** -19 * np.abs(qkv).max()).all()
        runs = plan.runs.to_storage()
        for i, (name, new) in enumerate((("k", y[:, Hq:]), ("v", qkv[:, Hq + Hkv:]))):
            codes, scale, refused = O.append(new, runs, form, before[i], before[2 + i], name == "v")
            same(getattr(cache, name).to_storage(), codes, name)
            same(getattr(cache, name + "_scale").to_storage(), scale, name + " scales")
        starts = plan.starts.to_storage()
        held = [x.to_storage() for x in (cache.k, cache.v, cache.k_scale, cache.v_scale)]
        want, spread, slip = O.attention(y[:, :Hq], tables.to_storage(), starts, total, form, *held, page, D ** -0.5)
        assert (np.abs(out - want) <= attention_bound(want, spread, slip, "bf16", D, 128)).all()
        lens, taken = plan.lens, plan.taken
    assert ops.index_errors() == 0 and taken.to_storage()[0] == sum(-(-t // page) for t in total)
