"""TreeAccept and KVKeep on the GPU against their restatement (oracle/draft_np.py),
whole state compared bit for bit; and steps of decoding that check drafts, from
the cache to the tokens and back."""
import numpy as np
import pytest

import accel_amd
from accel_amd import BF16, F16, F32, U32, KV_NONE
from oracle import draft_np, kvcache_np
from test_gpu_kv_pages import Both, narrow, widen
from test_gpu_paged_attention import as_type, bound, types
from test_gpu_tree_attention import trees

pytestmark = pytest.mark.gpu


def up(dev, x):
    x = np.ascontiguousarray(x, np.uint32)
    return dev.upload(x, U32) if x.size else accel_amd.Buffer(dev, 0, 0, U32, x.shape)


def run_accept(dev, tokens, parents, offsets, sampled, width, stream=None):
    n = len(offsets) - 1
    ins = [up(dev, x) for x in (tokens, parents, offsets, sampled)]
    outs = [up(dev, np.full(s, 55)) for s in ((n, width), (n,), (n,))]
    dev.TreeAccept(*ins, *outs, stream=stream)
    return ins, outs


def check_accept(dev, tokens, parents, offsets, sampled, width):
    *want, left_out = draft_np.accept(tokens, parents, offsets, sampled, width)
    ins, outs = run_accept(dev, tokens, parents, offsets, sampled, width)
    if left_out:
        with pytest.raises(accel_amd.AccelError, match="left out"):
            dev.sync()
    dev.sync()
    for b, w, name in zip(outs, want, ("path", "counts", "next")):
        assert np.array_equal(b.numpy(), w), name
    for b in ins + outs:
        b.free()
    return want


@pytest.mark.parametrize("kind", ["mixed", "chain", "star", "wide", "forest", "roots"])
@pytest.mark.parametrize("width", [1, 2, 7, 64, 65, 300, 4096])
def test_walks(dev, kind, width):
    rng = np.random.default_rng(width)
    nodes = [1, 0, 2, 63, 64, 65, 128, 200, 255, 256, 5, 0]
    off = np.concatenate([[0], np.cumsum(nodes)])
    par = trees(nodes, width, kind)
    T = len(par)
    # few tokens, so that walks go far and children share them
    for vocabulary in (1, 2, 3, 40):
        check_accept(dev, rng.integers(0, vocabulary, T), par, off,
                     rng.integers(0, vocabulary, T), width)


def test_walks_of_many_drafts(dev):
    rng = np.random.default_rng(0)
    nodes = rng.integers(0, 40, 3000)
    par = trees(nodes, 1)
    T = len(par)
    check_accept(dev, rng.integers(0, 3, T), par, np.concatenate([[0], np.cumsum(nodes)]),
                 rng.integers(0, 3, T), 12)


def test_walks_over_parents_and_tokens_of_no_sense(dev):
    rng = np.random.default_rng(2)
    nodes = [40, 300, 50, 7]
    off = np.concatenate([[0], np.cumsum(nodes)])
    T = int(off[-1])
    for high in (60, 1 << 32):
        check_accept(dev, rng.integers(0, 2, T), rng.integers(0, high, T), off,
                     rng.integers(0, 2, T), 20)
    # no token ends a walk, and is no draft's
    none = np.full(T, KV_NONE)
    want = check_accept(dev, none, trees(nodes, 0, "chain"), off, none, 5)
    assert want[1].tolist() == [1, 0, 1, 1]
    # offsets that do not ascend, or pass the rows, name what rows there are
    ins, outs = run_accept(dev, rng.integers(0, 2, 50), trees([50], 0), [0, 30, 10, 5000, 9],
                           rng.integers(0, 2, 50), 6)
    dev.sync()
    assert outs[1].numpy()[[1, 3]].tolist() == [0, 0] and (outs[1].numpy()[[0, 2]] >= 1).all()
    for b in ins + outs:
        b.free()


def test_no_drafts(dev):
    ins, outs = run_accept(dev, [], [], [0], [], 3)
    dev.sync()
    check_accept(dev, [], [], [0, 0, 0], [], 3)


# ---- keep ------------------------------------------------------------------------

class Keeps(Both):
    def keep(self, path, counts, nodes, seqs=None, stream=None):
        off = np.concatenate([[0], np.cumsum(nodes)]).astype(np.uint32)
        path = np.asarray(path, np.uint32)
        draft_np.keep(self.m, path, counts, off, seqs)
        self.dev.KVKeep(self.c, self.u32(path), self.u32(counts), self.u32(off), self.u32(seqs),
                        stream=stream)
        self.settle()


def some_path(rng, m, k, width):
    p = np.full(width, KV_NONE, np.uint32)
    p[:k] = np.sort(rng.permutation(m)[:k])
    return p


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("page,dim", [(8, 8), (8, 16), (16, 40), (32, 80), (64, 128), (8, 256),
                                      (256, 24)])
def test_keeps(dev, dtype, page, dim):
    rng = np.random.default_rng(page + dim)
    b = Keeps(dev, layers=3, pages=120, page=page, dim=dim, sequences=7, slots=max(3, 200 // page),
              dtype=dtype)
    for _ in range(4):
        nodes = rng.integers(0, 40, 7)
        b.reserve(nodes)
        counts = [int(rng.integers(0, min(m, 9) + 1)) for m in nodes]
        b.keep([some_path(rng, m, k, 9) for m, k in zip(nodes, counts)], counts, nodes)
    b.free()


@pytest.mark.parametrize("m,k", [(1, 0), (1, 1), (2, 1), (64, 64), (65, 63), (200, 130), (256, 200),
                                 (700, 300)])
def test_keeps_of_many_rows(dev, m, k):
    rng = np.random.default_rng(m)
    b = Keeps(dev, layers=1, pages=220, kv_heads=1, dim=40, sequences=2, slots=100)
    b.reserve([13, 5])
    b.reserve([m, 3])
    b.keep([some_path(rng, m, k, 300), some_path(rng, 3, 2, 300)], [k, 2], [m, 3])
    # all in place, and all but the first
    b.reserve([50, 50])
    b.keep([np.arange(50), np.arange(50)], [50, 20], [50, 50])
    b.reserve([50, 50])
    b.keep([np.arange(1, 50), np.arange(1, 50)], [49, 49], [50, 50])


def test_a_sequence_shortened_by_all_it_has(dev):
    b = Keeps(dev, sequences=4, pages=60, slots=14)
    b.reserve([100, 8, 0, 17])
    b.keep(np.zeros((4, 1)), [0, 0, 0, 0], [100, 8, 0, 1])
    assert b.m.lens.tolist() == [0, 0, 0, 16] and b.m.refs.sum() == 2
    b.reserve([30, 1, 9, 1])


def test_lists_and_padding(dev):
    rng = np.random.default_rng(3)
    b = Keeps(dev, sequences=6, pages=60, slots=9)
    b.reserve([30, 20, 10, 40, 5, 60])
    nodes, seqs = [10, 7, 12, 30], [5, KV_NONE, 1, 3]
    counts = [4, 3, 12, 6]
    b.keep([some_path(rng, m, k, 12) for m, k in zip(nodes, counts)], counts, nodes, seqs)


def test_what_cannot_be_kept_stays(dev):
    """Each with a neighbour that is served."""
    b = Keeps(dev, sequences=6, pages=60, slots=9)
    b.reserve([30, 20, 10, 40, 5, 60])
    good = [0, 3, 5, KV_NONE]
    for bad, count, m, seq in [
            ([0, 3, 3, 4], 4, 10, 0), ([3, 0, 4, 5], 2, 10, 0), ([0, 1, 2, 10], 4, 10, 0),
            ([0, KV_NONE, 0, 0], 2, 10, 0), ([0, 1, 2, 3], 5, 10, 0), ([0, 1, 2, 3], 4, 3, 0),
            ([0, 1, 2, 3], 0xffffffff, 10, 0), ([0, 1, 2, 3], 2, 31, 0), ([0, 1, 2, 3], 2, 8, 6),
            ([0, 1, 2, 3], 2, 8, KV_NONE - 1)]:
        before = b.m.lens.copy()
        b.keep([bad, good], [count, 3], [m, 8], [seq, 5])
        assert (b.m.lens == before - [0, 0, 0, 0, 0, 5]).all()
        b.reserve([5], [5])


def test_two_entries_of_one_sequence(dev):
    """One of the two is served, the other reported."""
    b = Keeps(dev, sequences=3, pages=30, slots=9)
    b.reserve([30, 20, 9])
    u = b.u32
    for _ in range(3):
        dev.KVKeep(b.c, u([[0, 1], [0, 2], [0, 1]]), u([2, 2, 1]), u([0, 5, 10, 13]), u([1, 1, 2]))
        with pytest.raises(accel_amd.AccelError, match="left out"):
            dev.sync()
        # either leaves the same lengths, pages and counts
        b.m.lens[1] -= 3
        b.m.lens[2] -= 2
        for s in (1, 2):
            for j in range(-(-int(b.m.lens[s]) // 8), 9):
                if b.m.tables[s, j] != KV_NONE:
                    b.m.refs[b.m.tables[s, j]] -= 1
                    b.m.tables[s, j] = KV_NONE
        for x in ("lens", "tables", "refs"):
            assert np.array_equal(getattr(b.c, x).numpy(), getattr(b.m, x)), x
        # what moved, if the second was served
        for x in ("keys", "values"):
            getattr(b.m, x)[:] = getattr(b.c, x).numpy()
        b.reserve([0, 0, 1])


def test_pages_that_another_sequence_has(dev):
    """Rows in shared pages may come from them and stay in them, not move into
    them; giving a shared page back leaves it to the others."""
    b = Keeps(dev, sequences=4, pages=60, slots=9)
    b.reserve([32, 0, 40, 0])
    b.fork([0, 2], [1, 3])
    b.keep([[0, 1, 5], [0, 1, 2]], [3, 3], [8, 8], [1, 0])     # pages 0 .. 3 shared: one may not
    assert b.m.lens.tolist() == [27, 32, 40, 40]
    b.keep([[0, 0, 0]], [0], [30], [3])
    assert b.m.lens[3] == 10
    b.reserve([0, 16, 0, 0])
    b.keep([[0, 1, 9]], [3], [16], [1])      # in pages of its own
    assert b.m.lens[1] == 35
    b.keep([[2, 3, 4]], [3], [11], [1])      # from its own into a shared one
    assert b.m.lens[1] == 35


def test_a_slot_without_a_page(dev):
    b = Keeps(dev, sequences=2, pages=30, slots=12)
    b.reserve([80, 80])
    b.trim(40)
    # positions 0 .. 39 are gone: rows move only where there are pages
    b.keep([[0, 60], [50, 60]], [2, 2], [75, 20], [0, 1])
    assert b.m.lens.tolist() == [80, 80]
    b.keep([[0, 1], [10, 12]], [2, 2], [75, 20], [0, 1])
    assert b.m.lens.tolist() == [7, 62]
    b.reserve([3, 3])


def test_keep_replays_and_streams(dev):
    """Captured once and replayed, other paths between the replays."""
    rng = np.random.default_rng(6)
    st = dev.stream()
    b = Keeps(dev, sequences=5, pages=80, slots=20)
    b.reserve([40, 10, 0, 25, 8])
    nodes = np.array([20, 9, 30, 12, 1], np.uint32)
    off = np.concatenate([[0], np.cumsum(nodes)]).astype(np.uint32)
    b.reserve(nodes)
    held = dict(path=b.u32(np.zeros((5, 6))), counts=b.u32(np.zeros(5)), off=b.u32(off))
    call = lambda: dev.KVKeep(b.c, held["path"], held["counts"], held["off"], stream=st)  # noqa: E731
    ex = None
    for i in range(5):
        counts = np.array([rng.integers(0, min(m, 6) + 1) for m in nodes], np.uint32)
        path = np.array([some_path(rng, m, k, 6) for m, k in zip(nodes, counts)])
        held["path"].write(path)
        held["counts"].write(counts)
        draft_np.keep(b.m, path, counts, off)
        if i == 1:
            dev.capture_begin(st)
            call()
            ex = dev.capture_end(st)
        dev.launch(ex, st) if ex else call()
        dev.sync(st)
        b.check()
        b.reserve(nodes - counts)
    dev.destroy_exec(ex)
    dev.destroy_stream(st)


# ---- together ----------------------------------------------------------------------

@types
def test_steps_of_checked_drafts(dev, q, kv):
    """Prompts, then steps that reserve, append and attend a draft's nodes in two
    layers, sample at each node from logits, walk, and keep: each step against its
    restatement, the cache's state bit for bit."""
    rng = np.random.default_rng(21)
    L, KV, H, D, P, B, V = 2, 2, 6, 40, 8, 3, 50
    c = dev.kv_cache(L, 60, KV, P, D, 4, 20, kv)
    m = kvcache_np.Pages(np.zeros((L, 60, KV, P, D), np.float32),
                         np.zeros((L, 60, KV, P, D), np.float32), 4, 20)
    u = lambda x: up(dev, x)  # noqa: E731
    seqs = [2, 0, 3]

    def rows(T):
        kr, vr = rng.standard_normal((2, T, KV, D)).astype(np.float32)
        return kr, vr

    def append(layer, off):
        kr, vr = rows(int(off[-1]))
        m.append(layer, widen(narrow(kr, kv), kv), widen(narrow(vr, kv), kv), seqs, off)
        dev.KVAppend(c, layer, dev.upload(kr), dev.upload(vr), u(seqs), u(off))

    first = [20, 7, 33]
    m.reserve(first, seqs)
    dev.KVReserve(c, u(first), u(seqs))
    for layer in range(L):
        append(layer, np.concatenate([[0], np.cumsum(first)]))
    for step in range(5):
        nodes = [int(x) for x in rng.integers(1, 14, B)]
        off = np.concatenate([[0], np.cumsum(nodes)]).astype(np.uint32)
        T = int(off[-1])
        par = trees(nodes, step)
        m.reserve(nodes, seqs)
        dev.KVReserve(c, u(nodes), u(seqs))
        for layer in range(L):
            append(layer, off)
            qv, qh = as_type(rng.standard_normal((T, H, D)) * 2, q)
            out = dev.alloc((T, H, D), q)
            dev.PagedTreeAttention(dev.upload(qh, q), u(off), u(par), c, out, layer=layer,
                                   seqs=u(seqs), window=25, sinks=2)
            dev.sync()
            got = out.numpy() if q == F32 else widen(out.numpy(), q)
            want, mass, size, _ = draft_np.attention(
                qv.astype(np.float64), m.keys[layer].astype(np.float64),
                m.values[layer].astype(np.float64), m.tables, m.lens, seqs, off, par,
                float(np.float32(D ** -0.5)), 25, 2)
            tol = bound(want, mass, size, q, kv, D, int(m.lens.max()), True)
            assert (np.abs(got - want) <= tol).all()
        x = (rng.standard_normal((T, V)) * 2).astype(np.float32)
        draws = rng.random(T).astype(np.float32)
        sampled, path, counts, nxt = (dev.upload(np.zeros(s, np.uint32))
                                      for s in ((T,), (B, 5), (B,), (B,)))
        dev.Sample(dev.upload(x), dev.upload(draws), sampled,
                   top_k=u(np.full(T, 6)), temperature=dev.upload(np.full(T, 0.8, np.float32)))
        want_s = [draft_np.sample(x[t], draws[t], float(np.float32(0.8)), 6)[0] for t in range(T)]
        # guesses that come true often
        draft = rng.integers(0, V, T)
        for i in range(B):
            for t in range(int(off[i]) + 1, int(off[i + 1])):
                if rng.random() < 0.6:
                    draft[t] = want_s[int(off[i]) + int(par[t])]
        dev.TreeAccept(u(draft), u(par), u(off), sampled, path, counts, nxt)
        dev.KVKeep(c, path, counts, u(off), u(seqs))
        wp, wc, wn, _ = draft_np.accept(draft, par, off, want_s, 5)
        draft_np.keep(m, wp, wc, off, seqs)
        dev.sync()
        assert sampled.numpy().tolist() == want_s
        for b, w in ((path, wp), (counts, wc), (nxt, wn), (c.lens, m.lens), (c.refs, m.refs),
                     (c.tables, m.tables)):
            assert np.array_equal(b.numpy(), w)
        for name in ("keys", "values"):
            held = widen(getattr(c, name).numpy(), kv)
            for s in seqs:
                for p in range(int(m.lens[s])):
                    pg = m.tables[s, p // P]
                    assert (held[:, pg, :, p % P] == getattr(m, name)[:, pg, :, p % P]).all()
    assert m.lens[seqs].sum() > sum(first) + 5 * B
    c.free()
