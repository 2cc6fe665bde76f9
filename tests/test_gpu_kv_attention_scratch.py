"""Attention over the paged cache: the scratch that both kinds of tiles share."""
import numpy as np
import pytest

from tests.kv_models import Batch, rows
from tests.test_gpu_kv_cache import check_attention

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("requests", [1, 2, 3, 4])
def test_scratch_of_both_kinds_begins_on_16_bytes(hip, requests):
    """Tables of 16384 tokens make the work of tiles of few columns and of many shared.  A request alone gives 33 workers to each of two heads for its few columns: 66 records of a tile's
    parts, in front of the sums of many columns (which the call refuses to write off 16 bytes)."""
    rng = np.random.default_rng(requests)
    b = Batch(rng, [300] + [70] * (requests - 1), [128] + [1] * (requests - 1), 64, 2, 128, "e4m3", table=256)
    check_attention(b, rows(rng, (b.N, 12, 128), "bf16"), "bf16", 12)
