"""The restatement of the paged cache (oracle/kvcache_np.py) where the header's
words decide (CPU)."""
import numpy as np

from oracle.kvcache_np import NONE, Pages


def pages(n, sequences, slots):
    shape = (1, n, 1, 8, 8)
    return Pages(np.zeros(shape, np.uint16), np.zeros(shape, np.uint16), sequences, slots)


def test_a_short_pool_serves_who_fits():
    m = pages(50, 5, 100)
    m.reserve([800, 1, 100, 0, 17])
    assert m.left_out == [0]
    assert list(m.lens) == [0, 1, 100, 0, 17]
    # the lowest free pages, as if the first entry were not there
    assert list(m.tables[1, :1]) == [0] and list(m.tables[2, :13]) == list(range(1, 14))
    assert list(m.tables[4, :3]) == [14, 15, 16]
    assert (m.tables[0] == NONE).all() and m.refs.sum() == 17
