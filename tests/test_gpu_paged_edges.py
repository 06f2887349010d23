"""The paged cache and its attention at the edges of what the header allows:
arguments near their types' ends, values that are not finite, queries and
scales that leave the normal range, weights far below the largest, a pool that
runs short.  Bounds are those of test_gpu_paged_attention.py unless said."""
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
