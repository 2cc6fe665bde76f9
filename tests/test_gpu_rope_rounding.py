"""Rotary positions: f32 rows are rounded once, like 16-bit ones."""
import numpy as np
import pytest

from oracle import kv_cache as O
from rai_amd import ops
from tests.kv_models import HALF_STEP, dev, rows
from tests.util import down, up

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("inverse", [False, True])
@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("far,magnitude", [(1, 1.0), (3000, 1.0), (3000, 1.2079), (10 ** 6, 1.2079)])
@pytest.mark.parametrize("shape,rot", [((257, 3, 128), 128), ((33, 14, 80), 32), ((65, 2, 256), 256), ((9, 5, 11), 6), ((40, 3, 72), 40)])
@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
def test_rounded_once(hip, dt, shape, rot, far, magnitude, inter, inverse):
    rng = np.random.default_rng(rot + far)
    x, p, f = rows(rng, shape, dt), rng.integers(0, far, shape[0]), O.frequencies(rot, 1e4)
    got = down(ops.rope_positions(up(x, dt), dev(p, "i64"), dev(f, "f64"), inter, inverse, magnitude)).astype(np.float64)
    want = O.rope(x, p, f, inter, inverse, magnitude)
    # Before the rounding.  f32 rows: an angle of up to `far` radians in f64, rounded four times (2^-53 of it each) here and in the oracle together, sines and cosines 2^-50, two
    # products and a sum 2^-51.  16-bit rows: the turn in f32 (2^-25 of half a turn, pi times that in the angle: 2^-23.3), sincospi and the magnitude 2^-22, two products and a sum 2^-23.
    other = np.abs(x) + np.abs(x).max(-1, keepdims=True)
    inner = far * 2.0 ** -51 + 2.0 ** -48 if dt == "f32" else 2.0 ** -21
    bound = HALF_STEP[dt] * (1 + 2.0 ** -6) * np.abs(want) + inner * magnitude * other + (2.0 ** -25 if dt == "f16" else 0)
    over = np.abs(got - want) / np.maximum(bound, 1e-300)
    assert (np.abs(got - want) <= bound).all(), f"{over.max()} of the bound, {np.mean(over > 1)} of the elements"
    if dt == "f32" and far == 3000:
        # a value is halfway between two f32 so rarely that all but a few are the nearest one
        assert np.mean(got != want.astype(np.float32)) < 1e-3
