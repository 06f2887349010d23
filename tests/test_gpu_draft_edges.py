"""Steps over drafts at their edges: what one does to the cache where something in it
cannot be served, whole steps as a graph, very many drafts; against the restatements
(oracle/draft_np.py, oracle/kvcache_np.py), the cache's state bit for bit."""
import numpy as np
import pytest

import accel_amd
from accel_amd import BF16, F32, U32, KV_NONE, NO_TOKEN
from oracle import draft_np, kvcache_np
from test_gpu_draft import Keeps, run_accept
from test_gpu_kv_pages import narrow, widen
from test_gpu_paged_attention import bound
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


def test_whole_steps_captured_and_replayed(dev):
    """Reserve, append, attention, sampling, walk and keep as one graph: other trees, rows,
    logits and guesses between the replays, a padded entry among them, eager work beside
    them; every step against its restatement."""
    rng = np.random.default_rng(30)
    st = dev.stream()
    L, KV, H, D, P, B, V, T, W = 2, 2, 4, 64, 8, 4, 300, 90, 6
    c = dev.kv_cache(L, 90, KV, P, D, 5, 30, BF16)
    m = kvcache_np.Pages(np.zeros((L, 90, KV, P, D), np.float32),
                         np.zeros((L, 90, KV, P, D), np.float32), 5, 30)
    first, seqs = [20, 7, 33, 0, 61], [2, 4, 0, 1]
    u = lambda x: dev.upload(np.asarray(x, np.uint32), U32)  # noqa: E731
    m.reserve(first)
    dev.KVReserve(c, u(first))
    for layer in range(L):
        kv = rng.standard_normal((2, sum(first), KV, D)).astype(np.float32)
        off = np.concatenate([[0], np.cumsum(first)]).astype(np.uint32)
        m.append(layer, *(widen(narrow(x, BF16), BF16) for x in kv), None, off)
        dev.KVAppend(c, layer, dev.upload(kv[0]), dev.upload(kv[1]), None, u(off))
    b = {k: u(np.zeros(n)) for k, n in dict(grow=B, off=B + 1, seqs=B, par=T, token=T, drawn=T,
                                            counts=B, next=B, top_k=T).items()}
    b["path"] = u(np.zeros((B, W)))
    for k, s in dict(k=(L, T, KV, D), v=(L, T, KV, D), q=(L, T, H, D), out=(L, T, H, D), x=(T, V),
                     u=(T,)).items():
        parts = s[0] if len(s) == 4 else 0
        b[k] = ([dev.upload(np.zeros(s[1:], np.float32)) for _ in range(parts)] if parts
                else dev.upload(np.zeros(s, np.float32)))

    def step():
        dev.KVReserve(c, b["grow"], b["seqs"], stream=st)
        for i in range(L):
            dev.KVAppend(c, i, b["k"][i], b["v"][i], b["seqs"], b["off"], stream=st)
            dev.PagedTreeAttention(b["q"][i], b["off"], b["par"], c, b["out"][i], layer=i,
                                   seqs=b["seqs"], window=30, sinks=3, stream=st)
        dev.Sample(b["x"], b["u"], b["drawn"], top_k=b["top_k"], stream=st)
        dev.TreeAccept(b["token"], b["par"], b["off"], b["drawn"], b["path"], b["counts"],
                       b["next"], stream=st)
        dev.KVKeep(c, b["path"], b["counts"], b["off"], b["seqs"], stream=st)

    ex, taken = None, 0
    for i in range(6):
        nodes = rng.integers(1, 20, B)
        off = np.concatenate([[0], np.cumsum(nodes)]).astype(np.uint32)
        n = int(off[-1])
        par = np.full(T, 999, np.uint32)
        par[:n] = trees(nodes, i, "wide" if i & 1 else "mixed")
        who = np.array(seqs, np.uint32)
        who[i % B] = KV_NONE if i == 3 else who[i % B]
        kv = rng.standard_normal((2, L, T, KV, D)).astype(np.float32)
        q = (rng.standard_normal((L, T, H, D)) * 2).astype(np.float32)
        x = (rng.standard_normal((T, V)) * 2).astype(np.float32)
        draws, top_k = rng.random(T).astype(np.float32), rng.integers(1, 9, T).astype(np.uint32)
        want_s = [draft_np.sample(x[t], draws[t], 1.0, top_k[t])[0] for t in range(T)]
        token = rng.integers(0, V, T).astype(np.uint32)
        for e in range(B):
            for t in range(int(off[e]) + 1, int(off[e + 1])):
                if rng.random() < 0.6:
                    token[t] = want_s[int(off[e]) + int(par[t])]
        for name, value in dict(grow=nodes.astype(np.uint32), off=off, seqs=who, par=par,
                                token=token, top_k=top_k, x=x, u=draws).items():
            b[name].write(value)
        for layer in range(L):
            b["k"][layer].write(kv[0, layer]), b["v"][layer].write(kv[1, layer])
            b["q"][layer].write(q[layer])
            b["out"][layer].write(np.full((T, H, D), 5, np.float32))
        if i == 1:
            dev.capture_begin(st)
            step()
            ex = dev.capture_end(st)
        dev.launch(ex, st) if ex else step()
        dev.sync(st)
        m.reserve(nodes, who)
        for layer in range(L):
            m.append(layer, *(widen(narrow(y[layer][:n], BF16), BF16) for y in kv), who, off)
            want, mass, size, left_out = draft_np.attention(
                q[layer].astype(np.float64), m.keys[layer].astype(np.float64),
                m.values[layer].astype(np.float64), m.tables, m.lens, who, off, par,
                float(np.float32(D ** -0.5)), 30, 3)
            tol = bound(want, mass, size, F32, BF16, D, int(m.lens.max()), True)
            got = b["out"][layer].numpy()
            assert not left_out and (np.abs(got - want) <= tol)[:n].all() and (got[n:] == 5).all()
        path, counts, nxt, _ = draft_np.accept(token, par, off, want_s, W)
        draft_np.keep(m, path, counts, off, who)
        assert b["drawn"].numpy().tolist() == want_s
        for got, want in ((b["path"], path), (b["counts"], counts), (b["next"], nxt),
                          (c.lens, m.lens), (c.refs, m.refs), (c.tables, m.tables)):
            assert np.array_equal(got.numpy(), want)
        assert not m.left_out
        taken += int(counts.sum())
        # eager work between the replays, on the same workspace
        dev.Sample(b["x"], b["u"], b["drawn"], stream=st)
        dev.sync(st)
    assert taken > 6 * B
    dev.destroy_exec(ex)
    dev.destroy_stream(st)
    c.free()


def test_more_drafts_than_a_launch_has_workgroups(dev):
    """A few more than 2^22 entries: walks of a node or two each, and keeps of which the
    first and the last have a sequence."""
    n = (1 << 22) + 7
    rng = np.random.default_rng(31)
    par = np.tile(np.array([KV_NONE, 0], np.uint32), n)
    token, drawn = (rng.integers(0, 2, 2 * n).astype(np.uint32) for _ in range(2))
    off = np.arange(0, 2 * n + 1, 2).astype(np.uint32)
    ins, outs = run_accept(dev, token, par, off, drawn, 2)
    dev.sync()
    takes = token[1::2] == drawn[::2]
    assert np.array_equal(outs[1].numpy(), 1 + takes)
    assert np.array_equal(outs[2].numpy(), np.where(takes, drawn[1::2], drawn[::2]))
    path = np.stack([np.zeros(n), np.where(takes, 1, KV_NONE)], 1)
    assert np.array_equal(outs[0].numpy(), path)
    b = Keeps(dev, pages=30, sequences=3, slots=9)
    b.reserve([20, 8, 30])
    seqs = np.full(n, KV_NONE, np.uint32)
    seqs[[0, n - 1]] = [2, 0]
    dev.KVKeep(b.c, outs[0], outs[1], ins[2], b.u32(seqs))
    ends = lambda x: x[[0, n - 1]]  # noqa: E731
    draft_np.keep(b.m, ends(path.astype(np.uint32)), ends(1 + takes), [0, 2, 4], [2, 0])
    b.settle()
    for x in ins + outs:
        x.free()
