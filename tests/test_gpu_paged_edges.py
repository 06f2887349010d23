"""The paged cache and its attention at the edges of what the header allows:
arguments near their types' ends, values that are not finite, queries and
scales that leave the normal range, weights far below the largest, a pool that
runs short.  Bounds are those of test_gpu_paged_attention.py unless said."""
import numpy as np
import pytest

from accel_amd import KV_NONE
from test_gpu_kv_pages import Both

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("window,sinks", [(1, 2 ** 63 - 1), (8, 2 ** 63 - 8), (1, 2 ** 31),
                                          (2 ** 63 - 1, 0), (2 ** 63 - 1, 2 ** 63 - 1)])
def test_trim_with_windows_and_sinks_past_any_table(dev, window, sinks):
    b = Both(dev, sequences=5, pages=60, slots=12)
    b.reserve([0, 1, 8, 64, 95])
    b.trim(window, sinks)
    assert (b.m.tables != KV_NONE).sum() == 22       # nothing is given back


def test_a_short_pool_serves_who_fits(dev):
    """An entry that the pool cannot serve takes nothing from those after it."""
    b = Both(dev, pages=50, sequences=8, slots=100)
    b.reserve([800, 1, 100, 0, 17], [0, 1, 2, 3, 4])
    assert list(b.m.lens[:5]) == [0, 1, 100, 0, 17]
    b.reserve([400, 9, 300, 3, 200, 1], [0, 1, 2, 3, 4, 5])
    b.reserve([8 * 50] * 8)
    b.reserve([0, 1, 8, 0, 1, 0, 8, 9])
    b.free([2])
    b.reserve([80, 16, 48, 16, 8, 8], [0, 2, 3, 5, 6, 7])


def test_a_short_pool_and_ever_smaller_entries(dev):
    """Needs that each pass what is left by one page, small ones between them."""
    n = 300
    b = Both(dev, layers=1, pages=n, kv_heads=1, page=8, dim=8, sequences=2 * n, slots=n + 1)
    b.reserve([8 * (1 if i % 2 == 0 else n - i // 2) for i in range(2 * n)])
    assert (b.m.lens[::2] != 0).sum() > n // 2


@pytest.mark.parametrize("seed", range(8))
def test_a_short_pool_of_many_entries(dev, seed):
    """More entries than the planning workgroup has lanes, pools within LDS and
    past it, in a mixed order with padding and repeated sequences."""
    rng = np.random.default_rng(seed)
    n, pages = [(40, 30), (1024, 300), (3000, 900), (3000, 5000)][seed % 4]
    b = Both(dev, layers=1, pages=pages, kv_heads=1, page=8, dim=8, sequences=n, slots=64)
    for _ in range(3):
        seqs = rng.permutation(n).astype(np.int64)
        seqs[rng.random(n) < 0.1] = KV_NONE
        seqs[rng.random(n) < 0.02] = int(seqs[0])
        grow = rng.integers(0, [60, 500, 20, 300][seed % 4], n)
        b.reserve([int(x) for x in grow], [int(s) for s in seqs])
        b.free([int(s) for s in rng.permutation(n)[:n // 3]])
