"""The 64-bit restatement of the paged 8-bit cache against torch's own conversions and plain formulas."""
import math

import numpy as np
import pytest
import torch

from oracle import kv_cache as O
from tests.kv_models import Batch


def test_codes_are_those_of_torch():
    every = np.arange(256, dtype=np.uint8)
    want = torch.from_numpy(every.copy()).view(torch.float8_e4m3fn).double().numpy()
    assert np.array_equal(O.values(every, "e4m3"), want, equal_nan=True)
    rng = np.random.default_rng(0)
    x = np.concatenate([rng.standard_normal(5000) * 10.0 ** rng.uniform(-4, 3, 5000), want[np.isfinite(want)], (want[:126] + want[1:127]) / 2, [0.0, -0.0, 1e9, -1e9]])
    x = np.clip(x.astype(np.float32), -448, 448)
    assert np.array_equal(O.codes(x, "e4m3"), torch.from_numpy(x).to(torch.float8_e4m3fn).view(torch.uint8).numpy())
    assert O.codes([np.nan, np.inf, -np.inf], "e4m3").tolist() == [0, 0x7e, 0xfe]
    assert O.codes([np.nan, np.inf, -np.inf, 0.5, 1.5, -126.6], "int8").view(np.int8).tolist() == [0, 127, -127, 0, 2, -127]


@pytest.mark.parametrize("form", ["e4m3", "int8"])
def test_scales_are_the_least_powers_that_hold(form):
    top = O.LARGEST[form]
    for e in (-99, -3, 0, 5, 100):
        assert O.scale_of(top * 2.0 ** e, form) == 2.0 ** e
        assert O.scale_of(np.nextafter(top * 2.0 ** e, np.inf), form) == 2.0 ** (e + 1)
    assert O.scale_of(0.0, form) == 2.0 ** -100 and O.scale_of(1e-40, form) == 2.0 ** -100
    assert O.scale_of(float(np.finfo(np.float32).max), form) == 2.0 ** O.MOST_EXP[form]


def test_plan_of_a_page_boundary_and_a_refusal():
    tables = np.array([[7, 0, 0], [9, 4, 0], [0, 0, 0]], np.uint32)
    got = O.plan([16, 20, 0], [1, 12, 33], np.array([1, 2, 3, 5], np.uint32), 1, tables, 16, 50, 50)
    t, lens, taken, starts, positions, runs, refused = got
    assert t.tolist() == [[7, 2, 0], [9, 4, 0], [0, 0, 0]] and lens.tolist() == [17, 32, 0] and taken == 2 and refused == 1
    assert starts.tolist() == [0, 1, 13, 46] and positions[:13].tolist() == [16] + list(range(20, 32)) and set(positions[13:].tolist()) == {-1}
    assert runs[:, :3].T.tolist() == [[2, 0, 0, 1], [4, 4, 1, 12], [0, 0, 0, 0]]


def test_rotation_is_a_complex_product():
    rng = np.random.default_rng(1)
    x, p, f = rng.standard_normal((5, 2, 10)), np.array([0, 1, 77, 10 ** 6, -1]), O.frequencies(8, 1e4)
    for inter in (False, True):
        pairs = np.stack([x[..., 0:8:2], x[..., 1:8:2]]) if inter else np.stack([x[..., :4], x[..., 4:8]])
        z = (pairs[0] + 1j * pairs[1]) * np.exp(1j * p[:, None, None] * f) * 1.5
        y = O.rope(x, p, f, inter, False, 1.5)
        got = y[..., 0:8:2] + 1j * y[..., 1:8:2] if inter else y[..., :4] + 1j * y[..., 4:8]
        assert np.allclose(got, z, rtol=0, atol=1e-12) and np.array_equal(y[..., 8:], x[..., 8:])
        # the gradient of sum(y g) is the turn back
        g = rng.standard_normal(x.shape)
        t = torch.tensor(x, requires_grad=True)
        a, b = (t[..., 0:8:2], t[..., 1:8:2]) if inter else (t[..., :4], t[..., 4:8])
        c, s = (torch.tensor(h(p[:, None, None] * f)) for h in (np.cos, np.sin))
        u, v = 1.5 * (a * c - b * s), 1.5 * (b * c + a * s)
        w = torch.tensor(g)
        ga, gb = (w[..., 0:8:2], w[..., 1:8:2]) if inter else (w[..., :4], w[..., 4:8])
        ((u * ga).sum() + (v * gb).sum() + (t[..., 8:] * w[..., 8:]).sum()).backward()
        assert np.allclose(O.rope(g, p, f, inter, True, 1.5), t.grad.numpy(), rtol=0, atol=1e-12)


def test_frequencies_blend_between_the_ends():
    f, s = O.frequencies(128, 5e5), O.frequencies(128, 5e5, 8.0, 1.0, 4.0, 8192)
    wave = 2 * math.pi / f
    assert np.array_equal(s[wave < 2048], f[wave < 2048]) and np.allclose(s[wave > 8192], f[wave > 8192] / 8)
    assert ((s <= f) & (s >= f / 8 * (1 - 1e-12))).all()


def test_attention_is_softmax_over_what_is_seen():
    rng = np.random.default_rng(2)
    b = Batch(rng, [5, 40, 3], [2, 1, 3], 16, 2, 24, "int8")
    q = rng.standard_normal((b.N, 4, 24))
    out, _, _ = O.attention(q, b.tables, b.starts, b.lens, "int8", b.k, b.v, b.k_scale, b.v_scale, 16, 0.2, window=7)
    k = O.values(b.k, "int8") * b.k_scale[:, :, None, None]
    v = O.values(b.v, "int8") * b.v_scale[:, :, None, None]
    keys = k[b.tables[1, :3], 1, :, :24].reshape(-1, 24)[33:40]
    vals = v[b.tables[1, :3], 1, :24].transpose(0, 2, 1).reshape(-1, 24)[33:40]
    w = torch.softmax(torch.tensor(q[2, 3] @ keys.T * 0.2), 0).numpy()
    assert np.allclose(out[2, 3], w @ vals, atol=1e-12)
    assert np.allclose(out[3, 0], v[b.tables[2, 0], 0, :24, 0], atol=1e-12)   # a prompt's first token sees itself
