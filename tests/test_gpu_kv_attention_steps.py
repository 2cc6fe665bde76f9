"""Attention over the paged cache where every step of 64 keys shows: each counted once, however the steps are dealt out and their parts joined."""
import numpy as np
import pytest

from tests import kv_steps
from tests.kv_models import dev
from tests.util import down, up


@pytest.mark.parametrize("dt", ["bf16", "f32"])
@pytest.mark.parametrize("name", kv_steps.CASES)
def test_a_step_too_few_or_too_many_would_show(name, dt):
    b, heads, window, scale, q = kv_steps.case(name, dt)
    assert kv_steps.least_seen(b, q, dt, heads, window, scale) > 3


@pytest.mark.gpu
@pytest.mark.parametrize("dt", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("name", kv_steps.CASES)
def test_every_step_counts_once(hip, name, dt):
    b, heads, window, scale, q = kv_steps.case(name, dt)
    got = down(b.cache().attention(up(q, dt), dev(b.tables, "u32"), dev(b.starts, "i64"), dev(b.lens, "i64"), scale, window)).astype(np.float64)
    want, bound = kv_steps.want(b, q, dt, scale, window)
    over = np.abs(got - want) / np.maximum(bound, 1e-300)
    assert (np.abs(got - want) <= bound).all(), f"{over.max()} of the bound at {np.unravel_index(over.argmax(), over.shape)}"
