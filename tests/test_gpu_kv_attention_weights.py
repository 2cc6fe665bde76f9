"""The softmax's weights in attention over the paged cache: of as many bits as the header says, in every kind of tile and whatever the width of the tables."""
import numpy as np
import pytest

from tests import kv_steps
from tests.kv_models import dev, rows
from tests.kv_steps import Seen
from tests.util import down, up

# more rows than tiles of few columns hold at once; the same for few rows, by the width of the tables alone; and tiles of few columns, tables near and wide
CASES = [([1] * 2, 12, 2, None), ([1] * 2, 12, 2, 2048), ([24], 12, 2, 8192), ([64] * 6, 40, 1, None), ([64, 1, 5], 40, 1, 4096)]


def batch(seed, dim, new, heads, kv, table, form):
    rng = np.random.default_rng(seed)
    return rng, Seen(rng, [dim - 3 * i for i in range(len(new))], new, 16, kv, dim, form, 1, table=table)


@pytest.mark.gpu
@pytest.mark.parametrize("dt", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("dim", [64, 80, 128, 256])
@pytest.mark.parametrize("new,heads,kv,table", CASES)
def test_weights_have_sixteen_bits(hip, new, heads, kv, table, dim, dt):
    for form in ("e4m3", "int8"):
        rng, b = batch(dim + heads, dim, new, heads, kv, table, form)
        q = rows(rng, (b.N, heads, dim), dt)
        got = down(b.cache().attention(up(q, dt), dev(b.tables, "u32"), dev(b.starts, "i64"), dev(b.lens, "i64"), dim ** -0.5)).astype(np.float64)
        want, bound = kv_steps.want(b, q, dt, dim ** -0.5)
        over = np.abs(got - want) / np.maximum(bound, 1e-300)
        assert (np.abs(got - want) <= bound).all(), f"{form}: {over.max()} of the bound, {np.mean(over > 1)} of the elements"


@pytest.mark.parametrize("dt", ["bf16", "f16", "f32"])
def test_the_bound_tells_weights_of_eight_bits(dt):
    """Each element here is one key's weight: with weights rounded to eight bits and all else exact, more than a hundred elements are outside."""
    import torch

    from oracle.dtypes import rnd
    for dim in (64, 256):
        rng, b = batch(dim, dim, [24], 12, 2, None, "e4m3")
        q = rows(rng, (b.N, 12, dim), dt)
        want, bound = kv_steps.want(b, q, dt, dim ** -0.5)
        # from the share of a key to the weight that a kernel holds, relative to its row's largest, and back
        top = want.max(-1, keepdims=True)
        weight = torch.from_numpy(want / top).to(torch.bfloat16).double().numpy() * top
        got = rnd(weight.astype(np.float32), dt).astype(np.float64)
        assert (np.abs(got - want) > bound).sum() > 100
        assert (np.abs(rnd(want.astype(np.float32), dt) - want) <= bound).all()
