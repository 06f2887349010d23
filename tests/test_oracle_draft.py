"""The restatement of drafts (oracle/draft_np.py) where the header's words decide
(CPU)."""
import math

import numpy as np
import pytest

from oracle import draft_np, kvcache_np
from oracle.draft_np import NONE


def test_a_chain_is_a_prompt():
    rng = np.random.default_rng(0)
    keys, values = rng.standard_normal((2, 9, 2, 8, 16))
    q = rng.standard_normal((7, 4, 16))
    tables = np.arange(9).reshape(1, 9).astype(np.uint32)
    lens = np.array([50], np.uint32)
    chain = np.array([NONE, 0, 1, 2, 3, 4, 5], np.uint32)
    for w, s in ((0, 0), (3, 2), (10, 45), (20, 0)):
        want = kvcache_np.attention(q, keys, values, tables, lens, [0], [0, 7], 0.3, w, s)
        got = draft_np.attention(q, keys, values, tables, lens, [0], [0, 7], chain, 0.3, w, s)
        assert got[3] == []
        for a, b in zip(want, got):
            assert np.allclose(a, b, rtol=1e-13, atol=0)


def test_a_branch_sees_its_own_line():
    rng = np.random.default_rng(1)
    keys, values = rng.standard_normal((2, 9, 1, 8, 8))
    q = rng.standard_normal((4, 1, 8))
    tables = np.arange(9).reshape(1, 9).astype(np.uint32)
    # 0 - 1, 0 - 2 - 3: node 3 without node 1 is a chain over a cache without it
    a = draft_np.attention(q, keys, values, tables, np.array([20]), [0], [0, 4],
                           [NONE, 0, 0, 2], 1.0, 5, 0)[0]
    k2, v2 = keys.copy(), values.copy()
    for x in (k2, v2):
        x[17 // 8, :, 17 % 8] = x[18 // 8, :, 18 % 8]
        x[18 // 8, :, 18 % 8] = x[19 // 8, :, 19 % 8]
    b = kvcache_np.attention(q[[0, 2, 3]], k2, v2, tables, np.array([19]), [0], [0, 3], 1.0, 5,
                             0)[0]
    assert np.allclose(a[[0, 2, 3]], b, rtol=1e-13, atol=0)


@pytest.mark.parametrize("kw,u,want", [
    (dict(), 0.0, 1), (dict(), 0.999999, 2), (dict(temperature=0.0), 0.9, 1),
    (dict(top_k=1), 0.99, 1), (dict(top_k=2), 0.9, 3), (dict(top_p=0.0), 0.9, 1),
    (dict(top_p=0.3), 0.99, 1), (dict(top_p=0.41), 0.99, 3), (dict(min_p=1.0), 0.9, 3),
    (dict(min_p=5.0), 0.9, 3), (dict(min_p=1.0), 0.1, 1), (dict(temperature=math.nan), 0.9, 1),
    (dict(top_p=math.nan), 0.99999, 2), (dict(), math.nan, 1), (dict(), 2.0, 2),
    (dict(temperature=math.inf), 0.3, 3), (dict(temperature=math.inf), 0.9, 2),
])
def test_tokens_by_hand(kw, u, want):
    # order: 1 and 3 (equal, 4/10 each), 0, 2 (1/10 each); 4 is not allowed, 5 no number
    x = [0.0, math.log(4), 0.0, math.log(4), -math.inf, math.nan]
    assert draft_np.sample(x, u, **kw)[0] == want


def test_tokens_of_rows_without_an_order():
    assert draft_np.sample([-math.inf, math.nan], 0.5)[:2] == (NONE, -math.inf)
    assert draft_np.sample([0.0, math.inf, 3.0, math.inf], 0.6)[0] == 3
    assert draft_np.sample([-0.0, 0.0], 0.4)[0] == 0


def test_a_walk_by_hand():
    parents = [NONE, 0, 0, 1, 1, 2, 9]
    tokens = [5, 7, 8, 1, 1, 2, 1]
    sampled = [7, 1, 9, 4, 6, 6, 6]
    path, counts, nxt, out = draft_np.accept(tokens, parents, [0, 7, 7], sampled, 5)
    assert path.tolist() == [[0, 1, 3, NONE, NONE], [NONE] * 5] and not out
    assert counts.tolist() == [3, 0] and nxt.tolist() == [4, NONE]
    path, counts, nxt, _ = draft_np.accept(tokens, parents, [0, 7], sampled, 2)
    assert path.tolist() == [[0, 1]] and counts[0] == 2 and nxt[0] == 1


def test_a_keep_by_hand():
    shape = (1, 6, 1, 8, 8)
    m = kvcache_np.Pages(np.arange(6 * 8 * 8).reshape(shape), np.zeros(shape), 2, 4)
    m.reserve([20, 9])
    was = m.keys.copy()
    draft_np.keep(m, [[0, 3, 5], [0, 0, 0]], [3, 0], [0, 9, 12])
    assert m.lens.tolist() == [14, 6] and m.refs.tolist() == [1, 1, 0, 1, 0, 0]
    assert (m.keys[0, 1, 0, 4] == was[0, 1, 0, 6]).all()          # 12 <- 14
    assert (m.keys[0, 1, 0, 5] == was[0, 2, 0, 0]).all()          # 13 <- 16
    assert m.left_out == []
    draft_np.keep(m, [[1, 1, 0], [3, 0, 0]], [2, 1], [0, 5, 8])
    assert m.left_out == [0, 1] and m.lens.tolist() == [14, 6]
