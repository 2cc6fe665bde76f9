"""Attention over the paged cache: keys whose values are zero, or far smaller than others', weigh like any."""
import numpy as np
import pytest

from tests import kv_steps
from tests.kv_models import Batch, dev, rows
from tests.util import down, up

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("new,heads,form", [([1, 1], 4, "e4m3"), ([1, 24], 40, "int8"), ([3, 24], 40, "e4m3")])
def test_pages_of_zeros(hip, new, heads, form):
    """One key above all the others by 19 (as a power of e), those in pages of zeros, whose scale is the least there is: together they weigh 5e-9 times their number."""
    rng = np.random.default_rng(heads)
    dt, total, page, dim = "f32", [120000, 110000], 64, 16
    b = Batch(rng, total, new, page, 1, dim, form, garbage=False)
    b.k[:], b.v[:], b.k_scale[:], b.v_scale[:] = 0, 0, 1.0, 2.0 ** -100
    one = 0x38 if form == "e4m3" else 1
    for r in range(2):
        p = b.tables[r, 100]
        b.k[p, 0, 7, 0] = one
        b.v[p, 0, 0, 7] = one
        b.v_scale[p] = 3.0
    q = rows(rng, (b.N, heads, dim), dt)
    q[..., 0] = 19.0
    got = down(b.cache().attention(up(q, dt), dev(b.tables, "u32"), dev(b.starts, "i64"), dev(b.lens, "i64"), 1.0)).astype(np.float64)
    want, _ = kv_steps.want(b, q, dt, 1.0)
    # counted out by hand for the last row of the first request
    last = b.starts[1] - 1
    assert np.allclose(want[last][:, 0], 3.0 / (1 + (total[0] - 1) * np.exp(-19.0)), rtol=1e-12)
    # a lane adds up sixteen weights of a step and then steps, of 64 keys each; the power of 2 has an argument of 28, rounded to 2^-20.  Without the zeros' weights: 6e-4.
    bound = np.abs(want) * (2 * (total[0] / 64 + 80) * 2.0 ** -24 + 2.0 ** -19)
    over = np.abs(got - want) / np.maximum(bound, 1e-300)
    assert (over[..., 0] <= 1).all() and (got[..., 1:] == 0).all(), f"{over[..., 0].max()} of the bound"
