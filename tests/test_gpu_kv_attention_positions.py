"""Attention over the paged cache: where rows sit, and what they see, in calls that go past a table or past the batch's rows."""
import numpy as np
import pytest

from oracle import kv_cache as O
from rai_amd import ops
from tests.kv_models import dev, rows
from tests.kv_steps import Seen, want
from tests.util import down, up

pytestmark = pytest.mark.gpu


def check(b, q, dt, scale, window=0):
    ops.index_errors()
    got = down(b.cache().attention(up(q, dt), dev(b.tables, "u32"), dev(b.starts, "i64"), dev(b.lens, "i64"), scale, window)).astype(np.float64)
    exact, bound = want(b, q, dt, scale, window)
    over = np.abs(got - exact) / np.maximum(bound, 1e-300)
    assert (np.abs(got - exact) <= bound).all(), f"{over.max()} of the bound at {np.unravel_index(over.argmax(), over.shape)}"
    return got


@pytest.mark.parametrize("window", [0, 1, 16, 100, 2 ** 31 - 1])
@pytest.mark.parametrize("more", [1, 5, 40, 150, 10 ** 12, 2 ** 62])
@pytest.mark.parametrize("dt,new,heads", [("bf16", [1, 9, 3], 8), ("f32", [9, 130, 1], 8), ("bf16", [130, 128, 60], 40)])
def test_a_length_past_the_table(hip, dt, new, heads, more, window):
    """Rows keep the positions that the length gives them, and see the tokens that the table holds."""
    rng = np.random.default_rng(heads + window % 1000)
    b = Seen(rng, [192, 160, 192], new, 16, 1, 64, "e4m3", 1, table=12)
    b.lens[:] = [192 + more, 160, 192 + more]
    got = check(b, rows(rng, (b.N, heads, 64), dt), dt, 0.1, window)
    assert ops.index_errors() == 2
    if 0 < window <= more - new[0]:
        assert (got[:new[0]] == 0).all()


@pytest.mark.parametrize("window", [0, 30])
@pytest.mark.parametrize("dt,heads", [("bf16", 8), ("f32", 40)])
@pytest.mark.parametrize("rows_there", [1, 39, 81, 100, 160, 199])
def test_requests_whose_rows_are_not_all_there(hip, rows_there, dt, heads, window):
    """As after a plan that refused requests for want of rows: starts go on past the batch's rows, and those that are there sit where they would."""
    rng = np.random.default_rng(rows_there + heads)
    b = Seen(rng, [200, 130, 190], [40, 40, 120], 16, 1, 64, "int8", 1, table=16)
    check(b, rows(rng, (rows_there, heads, 64), dt), dt, 0.1, window)
    assert ops.index_errors() == 0
    b.starts[3] = 2 ** 62
    b.lens[2] = 2 ** 62 + 3 - rows_there   # positions as far as numbers go
    check(b, rows(rng, (rows_there, heads, 64), dt), dt, 0.1, window)


@pytest.mark.parametrize("page", [16, 64])
@pytest.mark.parametrize("window", [1, 16, 50, 100])
@pytest.mark.parametrize("dt,heads,new", [("bf16", 8, [1, 1, 1]), ("f32", 8, [1, 33, 20]), ("bf16", 40, [110, 120, 30])])
def test_pages_that_a_window_has_left(hip, dt, heads, new, window, page):
    """Entries of pages that no row sees may be anything; those of pages of which a row would see one token count."""
    rng = np.random.default_rng(window + heads)
    b = Seen(rng, [400, 257, 300], new, page, 1, 64, "e4m3", 1)
    q = rows(rng, (b.N, heads, 64), dt)
    oldest = [t - n - window + 1 for t, n in zip(b.total, new)]
    for r, o in enumerate(oldest):
        b.tables[r, :o // page] = 2 ** 32 - 1 - np.arange(o // page)
    check(b, q, dt, 0.1, window)
    assert ops.index_errors() == 0
    for r in range(3):
        kept = b.tables[r, oldest[r] // page]
        b.tables[r, oldest[r] // page] = b.pages
        check(b, q, dt, 0.1, window)
        assert ops.index_errors() > 0, r
        b.tables[r, oldest[r] // page] = kept
