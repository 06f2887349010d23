"""What a step over drafts does to the cache where something in it cannot be served:
each call against its restatement (oracle/draft_np.py, oracle/kvcache_np.py), whole
state compared bit for bit."""
import numpy as np
import pytest

import accel_amd
from accel_amd import BF16, KV_NONE, NO_TOKEN
from oracle import draft_np
from test_gpu_draft import Keeps, run_accept
from test_gpu_tree_attention import Tree, trees

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("width", [1, 9, 300])
def test_a_draft_that_the_walk_refuses_is_left_by_the_keep(dev, width):
    """The walk's outputs go to the keep as they are: sequences whose draft is too large
    stay as they were, and the others are served."""
    rng = np.random.default_rng(width)
    nodes, seqs = [257, 9, 0, 300, 256], [0, 1, 2, 4, 5]
    off = np.concatenate([[0], np.cumsum(nodes)]).astype(np.uint32)
    b = Keeps(dev, pages=200, sequences=7, slots=60)
    b.reserve([40, 10, 21, 8, 33, 3, 50])
    b.reserve(nodes, seqs)
    before = b.m.lens.copy(), b.m.tables.copy()
    T = int(off[-1])
    token, par, drawn = rng.integers(0, 2, T), trees(nodes, 1), rng.integers(0, 2, T)
    ins, outs = run_accept(dev, token, par, off, drawn, width)
    dev.KVKeep(b.c, outs[0], outs[1], b.u32(off), b.u32(seqs))
    path, counts, nxt, refused = draft_np.accept(token, par, off, drawn, width)
    assert refused == [0, 3]
    draft_np.keep(b.m, path, counts, off, seqs)
    assert b.m.left_out == [0, 3]
    b.settle()
    for got, want in zip(outs, (path, counts, nxt)):
        assert np.array_equal(got.numpy(), want)
    assert nxt[0] == nxt[3] == NO_TOKEN
    for s in (0, 4):
        assert b.m.lens[s] == before[0][s] and (b.m.tables[s] == before[1][s]).all()
    assert b.m.lens[1] < before[0][1] and b.m.lens[2] == 21
    for x in ins + outs:
        x.free()


def test_a_count_of_zero_takes_back_more_than_a_draft(dev):
    """As the header says of it, whatever else the path holds."""
    b = Keeps(dev, pages=200, sequences=3, slots=60)
    b.reserve([20, 30, 40])
    b.reserve([300, 257, 5])
    b.keep([[KV_NONE, 7], [0, 0], [3, 2]], [0, 0, 0], [300, 257, 5])
    assert b.m.lens.tolist() == [20, 30, 40]


class Lives(Keeps):
    def append(self, layer, new, seqs, rows):
        off = np.concatenate([[0], np.cumsum(new)]).astype(np.uint32)
        shape = (int(off[-1]), self.m.keys.shape[2], self.m.keys.shape[4])
        k, v = (rows.integers(0, 1 << 14, shape).astype(np.uint16) for _ in range(2))
        self.m.append(layer, k, v, seqs, off)
        self.dev.KVAppend(self.c, layer, self.dev.upload(k, BF16), self.dev.upload(v, BF16),
                          self.u32(seqs), self.u32(off))
        self.settle()


def test_a_shortened_sequence_does_not_write_over_its_branch(dev):
    """A sequence that a keep ends inside a page that its branch has too: rows appended
    there would be the branch's, so they are left out and reported, those of the next
    pages and of other sequences stored.  As a branch of its own it grows."""
    rng = np.random.default_rng(4)
    b = Lives(dev, layers=2, pages=60, sequences=5, slots=9)
    b.reserve([32, 0, 10, 0, 0])
    b.fork([0], [1])
    b.keep([[0]], [0], [13], [0])                    # 19 left: the third page is both's
    assert b.m.lens.tolist() == [19, 32, 10, 0, 0]
    b.reserve([11, 0, 3, 0, 0])
    held = b.m.keys[:, b.m.tables[1, 2]].copy()
    for layer in range(2):
        b.m.left_out = []
        b.append(layer, [11, 3], [0, 2], rng)
    assert (b.m.keys[:, b.m.tables[1, 2]] == held).all()
    # positions 24 to 29 lie in a page of its own
    b.append(0, [6], [0], rng)
    b.keep([[0]], [0], [11], [0])
    b.fork([0], [3])
    b.free([0])
    b.reserve([0, 0, 0, 12, 0])
    for layer in range(2):
        b.append(layer, [12], [3], rng)
    # and so does a sequence whose branch is gone
    b.keep([[0]], [0], [5], [1])
    b.fork([1], [4])
    b.free([4])
    b.reserve([0, 4, 0, 0, 0])
    b.append(1, [4], [1], rng)


@pytest.mark.parametrize("n", [1025, 2100, 4200])
def test_more_drafts_than_a_pass_over_them(dev, n):
    """Their steps are summed up 1024 at a time, and found again 64 ways a step: twice
    past 4096."""
    rng = np.random.default_rng(n)
    new = [int(x) for x in rng.integers(0, 4, n)]
    c = Tree(dev, [int(m + x) for m, x in zip(new, rng.integers(0, 12, n))], new, heads=2,
             kv_heads=1, dim=16, page=8)
    c.check()
    c.check(window=5, sinks=1)
