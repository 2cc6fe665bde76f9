"""Serving over the paged cache with nothing to do: steps without rows, tables without pages."""
import numpy as np
import pytest

from rai_amd import ops
from rai_amd.hip import HipTensor
from rai_amd.kv_cache import KvCache
from tests.kv_models import dev, rows
from tests.util import down, up

pytestmark = pytest.mark.gpu


def test_a_step_in_which_every_request_pauses(hip):
    rng = np.random.default_rng(1)
    cache = KvCache(8, 2, 64, 16, "e4m3")
    tables = dev(rng.permutation(8).astype(np.uint32).reshape(2, 4), "u32")
    before = [t.to_storage() for t in (tables, cache.k, cache.v, cache.k_scale, cache.v_scale)]
    ops.index_errors()
    plan = ops.kv_plan(dev(np.array([17, 0], np.int64), "i64"), dev(np.zeros(2, np.int64), "i64"), dev(np.zeros(0, np.uint32), "u32"), dev(np.zeros(1, np.int64), "i64"), tables, 16, 0)
    assert plan.lens.to_storage().tolist() == [17, 0] and plan.starts.to_storage().tolist() == [0, 0, 0] and plan.taken.to_storage().tolist() == [0]
    assert plan.positions.shape == (0,) and plan.runs.shape == (4, 0)
    nothing = HipTensor.empty((0, 2, 64), "bf16")
    turned = ops.rope_positions(nothing, plan.positions, ops.rope_frequencies(64, 1e4))
    cache.append(turned, nothing, plan.runs)
    assert cache.attention(HipTensor.empty((0, 8, 64), "bf16"), tables, plan.starts, plan.lens, 0.1).shape == (0, 8, 64)
    for t, b in zip((tables, cache.k, cache.v, cache.k_scale, cache.v_scale), before):
        assert np.array_equal(t.to_storage(), b)
    assert ops.index_errors() == 0


@pytest.mark.parametrize("lens,errors", [([0, 0], 0), ([5, 0], 1)])
@pytest.mark.parametrize("heads", [8, 40])
def test_tables_of_no_pages(hip, heads, lens, errors):
    rng = np.random.default_rng(2)
    cache = KvCache(3, 1, 64, 16, "int8")
    ops.index_errors()
    q = up(rows(rng, (300, heads, 64), "bf16"), "bf16")
    got = down(cache.attention(q, HipTensor.empty((2, 0), "u32"), dev(np.array([0, 290, 300], np.int64), "i64"), dev(np.array(lens, np.int64), "i64"), 0.1))
    assert (got == 0).all() and ops.index_errors() == errors
