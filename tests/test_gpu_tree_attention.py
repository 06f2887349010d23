"""PagedTreeAttention on the GPU against attention in 64 bits from its definition
(oracle/draft_np.py), within the bounds of test_gpu_paged_attention.py: the
products, the softmax and the roundings are those of a prompt's rows."""
import numpy as np
import pytest

import accel_amd
from accel_amd import BF16, F16, F32, U32, KV_NONE
from oracle import draft_np
from test_gpu_kv_pages import narrow, widen
from test_gpu_paged_attention import Case, bound, types

pytestmark = pytest.mark.gpu


def trees(nodes, seed=0, kind="mixed"):
    """Each entry's parents, in its own numbers."""
    rng = np.random.default_rng(seed)
    out = []
    for m in nodes:
        t = np.arange(m)
        up = {"mixed": (rng.random(m) * t).astype(np.int64), "chain": t - 1,
              "star": np.zeros(m, np.int64), "wide": (t - 1) // 3,
              "forest": np.where(rng.random(m) < 0.3, -1, (rng.random(m) * t).astype(np.int64)),
              "roots": np.full(m, -1)}[kind].copy()
        up[:1] = -1
        out.append(np.where(up < 0, KV_NONE, up))
    return np.concatenate(out + [np.zeros(0)]).astype(np.uint32)


class Tree(Case):
    """A cache of `lens` positions, the last new[i] of them an entry's nodes."""

    def __init__(self, dev, lens, new, parents=None, kind="mixed", **kw):
        super().__init__(dev, lens, new=new, **kw)
        if parents is None:
            parents = trees(new, kw.get("seed", 0), kind)
        # rows that no entry covers have parents of no sense
        self.parents = np.full(self.T, 12345, np.uint32)
        self.parents[:len(parents)] = parents

    def upload(self):
        super().upload()
        self.par_b = self.dev.upload(self.parents, U32)

    def call(self, layer=0, scale=0.0, window=0, sinks=0, stream=None):
        self.dev.PagedTreeAttention(self.qb, self.off_b, self.par_b, self.cache, self.out,
                                    layer=layer, seqs=self.seqs_b, scale=scale, window=window,
                                    sinks=sinks, stream=stream)

    def want(self, layer=0, scale=0.0, window=0, sinks=0):
        scale = scale or float(np.float32(self.dim ** -0.5))
        *r, self.oracle_left_out = draft_np.attention(
            self.q.astype(np.float64), self.k[layer].astype(np.float64),
            self.v[layer].astype(np.float64), self.tables, self.lens, self.seqs, self.off,
            self.parents, scale, window, sinks)
        return r

    def free(self):
        super().free()
        self.par_b.free()


@types
@pytest.mark.parametrize("m", [1, 2, 3, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 255, 256])
def test_nodes(dev, q, kv, m):
    Tree(dev, [70 + m], [m], q=q, kv=kv, seed=m).check()


@types
@pytest.mark.parametrize("before", [0, 1, 31, 32, 33, 63, 64, 65, 100, 127, 128, 1000])
def test_contexts(dev, q, kv, before):
    Tree(dev, [before + 20, before + 70], [20, 70], q=q, kv=kv, seed=before).check()


@types
@pytest.mark.parametrize("kind", ["chain", "star", "wide", "forest", "roots"])
def test_shapes_of_trees(dev, q, kv, kind):
    Tree(dev, [130, 50, 256, 7], [100, 50, 256, 1], q=q, kv=kv, kind=kind).check()


@types
@pytest.mark.parametrize("dim", [8, 24, 64, 80, 96, 120, 128, 136, 192, 256])
def test_head_dims(dev, q, kv, dim):
    Tree(dev, [90, 41], [33, 13], dim=dim, q=q, kv=kv, seed=dim).check()


@types
@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (3, 1), (4, 4), (6, 3), (7, 1), (16, 1),
                                            (17, 1), (40, 1), (130, 1), (32, 8)])
def test_groups(dev, q, kv, heads, kv_heads):
    Tree(dev, [85, 150], [45, 10], heads=heads, kv_heads=kv_heads, q=q, kv=kv, seed=heads).check()


@pytest.mark.parametrize("q,kv", [(F32, F16), (BF16, BF16)])
@pytest.mark.parametrize("n", [2, 66])
def test_more_heads_than_workgroups(dev, q, kv, n):
    """A key-value head's whole line is one workgroup's then, and none of it is cut."""
    nodes = [5, 33] if n == 2 else [3] * 65 + [40]
    Tree(dev, [m + 30 + i % 7 for i, m in enumerate(nodes)], nodes, heads=600, kv_heads=600,
         dim=8, q=q, kv=kv).check(window=0 if n == 2 else 20)


@pytest.mark.parametrize("page", [8, 16, 32, 64, 128, 4096])
def test_pages(dev, page):
    Tree(dev, [page + 9, 2 * page, 40], [9, 30 if page > 8 else 16, 40], page=page,
         seed=page).check()


@types
@pytest.mark.parametrize("kind", ["chain", "mixed", "forest"])
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (2, 0), (16, 0), (17, 4), (64, 4),
                                          (5, 200), (5, 75), (10000, 3), (1 << 40, 7)])
def test_window_and_sinks(dev, q, kv, kind, window, sinks):
    Tree(dev, [230, 64, 300, 40], [100, 20, 17, 40], q=q, kv=kv, kind=kind).check(
        window=window, sinks=sinks)


def test_window_over_pages_given_back(dev):
    c = Tree(dev, [700, 300], [100, 40], kind="wide")
    for i, (n, new) in enumerate([(700, 100), (300, 40)]):
        for j in range(c.tables.shape[1]):
            if j * 16 >= 5 and (j + 1) * 16 <= n - new - 50 + 1:
                c.tables[i, j] = KV_NONE
    c.check(window=50, sinks=5)


def test_padding_empty_entries_and_rows_behind(dev):
    Tree(dev, [40, 7, 100, 30], [40, 5, 0, 64, 0, 9], seqs=[0, KV_NONE, 1, 2, 3, 3],
         extra_rows=21).check()


def test_many_entries(dev):
    rng = np.random.default_rng(9)
    new = [int(x) for x in rng.integers(0, 12, 300)]
    Tree(dev, [int(n + x) for n, x in zip(new, rng.integers(0, 40, 300))], new, heads=2,
         kv_heads=1, dim=16, page=8).check()


def test_layers_and_scale(dev):
    c = Tree(dev, [90, 70], [40, 11], layers=3)
    for layer in range(3):
        c.check(layer=layer, scale=0.05 * (layer + 1))


@types
@pytest.mark.parametrize("window,sinks", [(0, 0), (1500, 30)])
def test_few_nodes_after_a_long_context(dev, q, kv, window, sinks):
    """Tiles of rows that several workgroups share, joined in a fixed order."""
    c = Tree(dev, [3000, 700, 2100, 0], [5, 64, 1, 0], heads=4, kv_heads=2, q=q, kv=kv)
    c.check(window=window, sinks=sinks)
    c.upload()
    first = None
    for _ in range(4):
        c.call(window=window, sinks=sinks)
        dev.sync()
        got = c.out.numpy()
        assert first is None or np.array_equal(first, got)
        first = got
    c.free()


@types
def test_uneven_contexts(dev, q, kv):
    lens = [40, 3000, 5, 900, 64, 1, 2000, 129]
    new = [8, 30, 5, 64, 64, 1, 3, 100]
    Tree(dev, lens, new, heads=8, kv_heads=2, dim=128, q=q, kv=kv).check()


# ---- what is reported ------------------------------------------------------------

@pytest.mark.parametrize("bad", [5, 6, 299, KV_NONE - 1], ids=["itself", "past", "far", "huge"])
def test_a_parent_that_is_not_before_its_child(dev, bad):
    """The node and those behind it are zeros, the rest is served."""
    c = Tree(dev, [100, 60], [40, 10], kind="wide")
    c.parents[5] = bad
    c.left_out = True
    c.check()
    assert {x[0] for x in c.oracle_left_out} == {"row"} and len(c.oracle_left_out) > 3
    c.check(window=9, sinks=2)


def test_entries_too_large_or_longer_than_their_sequence(dev):
    c = Tree(dev, [400, 20, 50, 90], [257, 30, 10, 9], seqs=[0, 1, 2, 7])
    c.left_out = True
    c.check()
    assert c.oracle_left_out == [("entry", 0), ("entry", 1), ("entry", 3)]


def test_bad_pages_are_left_out(dev):
    c = Tree(dev, [100, 100, 64], [50, 20, 64])
    c.tables[0, 2] = 0x7fffffff
    c.tables[1, :] = KV_NONE
    c.tables[2, 1] = KV_NONE             # among the nodes' own
    c.left_out = True
    c.check()


@pytest.mark.parametrize("n", [64, 100])
def test_entries_that_share_rows_past_32_bits_of_work(dev, n):
    """Offsets that do not ascend: 8 tiles of rows against 2^24 tiles of keys, so often
    that their number passes 32 bits.  No step of it is taken."""
    page, slots = 4096, 1 << 18
    u = lambda x: dev.upload(np.asarray(x, np.uint32), U32)  # noqa: E731
    c = dev.kv_cache(1, 1, 1, page, 8, 1, slots)
    c.lens.write(np.array([page * slots], np.uint32))
    off = np.zeros(n + 1, np.uint32)
    off[1::2] = 256
    q = dev.upload(np.zeros((256, 4, 8), np.uint16), BF16)
    out = dev.upload(np.full((256, 4, 8), 77, np.uint16), BF16)
    dev.PagedTreeAttention(q, u(off), u(trees([256])), c, out, seqs=u(np.zeros(n)))
    with pytest.raises(accel_amd.AccelError, match="draft's parents"):
        dev.sync()
    assert (out.numpy() == 77).all()
    c.free()


def test_a_report_is_read_once(dev):
    c = Tree(dev, [100], [40])
    c.parents[7] = 7
    c.upload()
    c.call()
    with pytest.raises(accel_amd.AccelError, match="draft's parents"):
        dev.sync()
    dev.sync()
    c.free()


# ---- numbers that are not finite, and large ones -----------------------------------

@types
def test_extreme_scores(dev, q, kv):
    Tree(dev, [140], [60], q=q, kv=kv, gain=60.0).check()
    c = Tree(dev, [140], [60], q=q, kv=kv)
    c.q[:], c.qh[:] = 0, 0
    c.check()
    Tree(dev, [140], [60], q=q, kv=kv, gain=1e-4, kv_gain=1e-3).check()
    Tree(dev, [140], [60], q=q, kv=kv, gain=1e-3, kv_gain=2e3).check()


@types
@pytest.mark.parametrize("bits", ["inf", "-inf", "nan"])
@pytest.mark.parametrize("lost", [False, True])
def test_values_that_are_not_finite_reach_only_who_sees_them(dev, q, kv, bits, lost):
    """A context's value and a node's value and key are not finite: nodes of other
    branches, and of windows past them, are what they were; and so are zeros."""
    x = {"inf": np.inf, "-inf": -np.inf, "nan": np.nan}[bits]
    b = narrow(np.array([x], np.float32), kv)[0]
    for window, sinks in ((0, 0), (40, 3)):
        c = Tree(dev, [250], [120], kind="wide", q=q, kv=kv, heads=4, kv_heads=2, dim=64)
        if lost:
            c.parents[100] = 110
        L = 130
        at = lambda j: (c.tables[0, j // 16], slice(None), j % 16)  # noqa: E731
        early, value, key = 92, L + 4, L + 7
        if window:
            c.vh[0][at(early)][:, 3:60:7] = b
        c.vh[0][at(value)][:, 3:60:7] = b
        c.kh[0][at(key)][:, 9] = b
        c.upload()
        c.call(window=window, sinks=sinks)
        if lost:
            with pytest.raises(accel_amd.AccelError, match="left out"):
                dev.sync()
        dev.sync()
        got = c.got()
        want, mass, size = c.want(window=window, sinks=sinks)
        tol = bound(want, mass, size, q, kv, 64, 250, True)
        lines = [draft_np.line_of(c.parents, t) for t in range(120)]
        depth = np.array([len(l) - 1 if l else -1 for l in lines])
        on = lambda a: np.array([bool(l) and a in l for l in lines])  # noqa: E731
        sees_early = (depth >= 0) & (L + depth - early < window) if window else depth > 999
        sees_value, sees_key = on(4), on(7)
        clean = ~sees_early & ~sees_value & ~sees_key
        assert clean.sum() >= 10 and sees_value.any() and sees_key.any()
        assert (np.abs(got - want) <= tol)[clean].all()
        shows = (sees_early | sees_value) & ~sees_key
        cols = np.zeros(64, bool)
        cols[3:60:7] = True
        assert not np.isfinite(got[shows][..., cols]).any()
        if not (bits == "nan"):
            assert (got[shows][..., cols] == x).all()
        assert (np.abs(got - want) <= tol)[shows][..., ~cols].all()
        if bits == "nan":
            assert np.isnan(got[sees_key]).all()
        c.free()


# ---- streams, graphs, large caches ---------------------------------------------------

def test_replays_and_streams(dev):
    """Captured once on a stream of its own and replayed, lengths and trees changing
    between the replays, beside another captured call on the same workspace."""
    st = dev.stream()
    a = Tree(dev, [3000, 500], [3, 70], heads=8, kv_heads=2, dim=128, q=F32)
    b = Tree(dev, [900], [40], heads=4, kv_heads=1, seed=3)
    execs = []
    for c in (a, b):
        c.upload()
        c.call(stream=st)
        dev.sync(st)
        c.compare()
        dev.capture_begin(st)
        c.call(stream=st)
        execs.append(dev.capture_end(st))
    for n, kind in ((2999, "chain"), (100, "star"), (3, "wide"), (3000, "roots")):
        a.lens[0] = n
        a.cache.lens.write(a.lens)
        a.parents[:] = trees([3, 70], n, kind)
        a.par_b.write(a.parents)
        for c, ex in ((a, execs[0]), (b, execs[1])):
            c.out.write(c.fill)
            dev.launch(ex, st)
            dev.sync(st)
            c.compare()
    for ex in execs:
        dev.destroy_exec(ex)
    for c in (a, b):
        c.free()
    dev.destroy_stream(st)


def test_a_chain_is_a_prompt(dev):
    """A tree without branches gives what PagedPrefill gives, within both bounds."""
    for q, kv in ((BF16, BF16), (F32, F16)):
        a = Tree(dev, [700, 90], [60, 33], kind="chain", q=q, kv=kv, heads=8, kv_heads=2, dim=128)
        a.upload()
        a.call(window=200, sinks=3)
        dev.sync()
        tree = a.got()
        a.out.write(a.fill)
        Case.call(a, window=200, sinks=3)
        dev.sync()
        want, mass, size = a.want(window=200, sinks=3)
        tol = bound(want, mass, size, q, kv, 128, 700, True)
        assert (np.abs(tree - a.got()) <= 2 * tol).all()
        a.free()


def test_keys_far_apart_in_a_large_cache(dev):
    """Offsets past 32 bits: the last pages of layer 1 of 2.3e9 elements a plane
    give what the first pages of a small cache give, bit for bit."""
    rng = np.random.default_rng(2)
    KV, P, D, H, n = 8, 256, 256, 16, 700
    k, v = (rng.standard_normal((n, KV, D)).astype(np.float32) for _ in range(2))
    q = narrow(rng.standard_normal((40, H, D)).astype(np.float32) * 2, BF16)
    u = lambda x: dev.upload(np.asarray(x, np.uint32), U32)  # noqa: E731
    par = trees([40], 5)
    res = []
    for layers, pages, before in ((2, 2200, 2197), (1, 3, 0)):
        c = dev.kv_cache(layers, pages, KV, P, D, 2, 2200)
        if before:
            dev.KVReserve(c, u([before * P]), u([1]))
        dev.KVReserve(c, u([n]), u([0]))
        dev.KVAppend(c, layers - 1, dev.upload(k), dev.upload(v), u([0]), u([0, n]))
        out, path = dev.alloc((40, H, D), BF16), np.full((1, 9), KV_NONE, np.uint32)
        dev.PagedTreeAttention(dev.upload(q, BF16), u([0, 40]), u(par), c, out, layer=layers - 1,
                               seqs=u([0]))
        dev.sync()
        path[0, :5] = [0, 3, 4, 20, 39]
        dev.KVKeep(c, u(path), u([5]), u([0, 40]), seqs=u([0]))
        after = dev.alloc((1, H, D), BF16)
        dev.PagedAttention(dev.upload(q[:1], BF16), c, after, layer=layers - 1, seqs=u([0]))
        dev.sync()
        assert c.tables.numpy()[0, 0] == before and c.lens.numpy()[0] == n - 35
        res.append((out.numpy(), after.numpy()))
        c.free()
    for a, b in zip(*res):
        assert np.array_equal(a, b) and np.isfinite(widen(a, BF16)).all()
