"""The paged cache's bookkeeping and its pages' moves on the GPU against the
list-by-list restatement (oracle/kvcache_np.py): whole state compared bit for
bit after every call, what cannot be served left out and reported."""
import numpy as np
import pytest

import accel_amd
from accel_amd import BF16, F16, F32, U32, KV_NONE
from oracle.kvcache_np import Pages

pytestmark = pytest.mark.gpu


class Both:
    """One cache on the device and its restatement."""

    def __init__(self, dev, layers=2, pages=40, kv_heads=2, page=8, dim=16, sequences=6, slots=9,
                 dtype=BF16, seed=0):
        rng = np.random.default_rng(seed)
        shape = (layers, pages, kv_heads, page, dim)
        k, v = (rng.integers(0, 1 << 16, shape).astype(np.uint16) for _ in range(2))
        self.dev, self.m = dev, Pages(k, v, sequences, slots)
        self.c = dev.kv_cache(layers, pages, kv_heads, page, dim, sequences, slots, dtype)
        self.c.keys.write(k)
        self.c.values.write(v)
        self.check()

    def u32(self, x):
        return None if x is None else self.dev.upload(np.asarray(x, np.uint32), U32)

    def check(self):
        for name in ("refs", "tables", "lens", "keys", "values"):
            got = getattr(self.c, name).numpy()
            want = getattr(self.m, name)
            assert np.array_equal(got, want), (name, np.argwhere(got != want)[:5])
        # what the counts stand for
        t = self.m.tables
        assert np.array_equal(np.bincount(t[t != KV_NONE], minlength=self.m.pages), self.m.refs)

    def settle(self, words=None):
        """The call's report: one where the restatement left entries out."""
        if self.m.left_out:
            with pytest.raises(accel_amd.AccelError, match="left out"):
                self.dev.sync()
        self.dev.sync()
        self.m.left_out = []
        self.check()

    def reserve(self, grow, seqs=None):
        self.m.reserve(grow, seqs)
        self.dev.KVReserve(self.c, self.u32(grow), self.u32(seqs))
        self.settle()

    def fork(self, parents, children):
        self.m.fork(parents, children)
        self.dev.KVFork(self.c, self.u32(parents), self.u32(children))
        self.settle()

    def free(self, seqs=None):
        self.m.free(seqs)
        self.dev.KVFree(self.c, self.u32(seqs))
        self.settle()

    def trim(self, window, sinks=0, seqs=None):
        self.m.trim(window, sinks, seqs)
        self.dev.KVTrim(self.c, window, sinks, self.u32(seqs))
        self.settle()

    def compact(self):
        want = self.m.compact()
        live = self.dev.upload(np.array([77], np.uint32))
        self.dev.KVCompact(self.c, live)
        self.settle()
        assert live.numpy()[0] == want

    def copy(self, src, dst):
        self.m.copy(src, dst)
        self.dev.KVCopy(self.c, self.u32(src), self.u32(dst))


def test_a_life_of_a_cache(dev):
    b = Both(dev)
    b.reserve([9, 0, 16, 1, 7, 8])                  # all sequences, one of them nothing
    b.reserve([7, 1, 30], [0, 1, 5])                # a list, in its order
    b.fork([0, 5, 0], [3, 1, 2])                    # 3, 1 and 2 are not empty: left out
    b.free([3, 1])
    b.fork([5, 0], [1, 3])                          # a partly full last page, and none
    b.reserve([1, 1, 1, 1, 1, 1])                   # branches grow apart
    b.trim(8, 3, [5])
    b.trim(1)
    b.free([5, 5, 2, KV_NONE])                      # one of them named twice
    b.compact()
    b.reserve([20, 20], [2, 5])
    b.compact()
    b.free()
    b.compact()


@pytest.mark.parametrize("page", [8, 16, 64])
def test_growth_by_whole_and_partial_pages(dev, page):
    b = Both(dev, page=page, pages=64, slots=12)
    for grow in (1, page - 1, page, page + 1, 3 * page, 0):
        b.reserve([grow] * 6)


def test_no_room(dev):
    b = Both(dev, pages=10, slots=4)
    b.reserve([33, 32, 1], [0, 1, 2])               # 0: more than its slots hold
    b.reserve([16, 20, 8], [3, 4, 5])               # 4 and those after it find no page
    b.reserve([0, 7], [5, 2])                       # growth inside a page needs none
    b.reserve([8, 8], [0, 0])                       # named twice
    b.reserve([1, 1, 1], [6, KV_NONE, 0xfffffff0])  # outside the cache; padding
    b.reserve([0xffffffff], [1])                    # does not wrap around
    b.free([2])
    b.fork([0, 0, 1], [2, 5, 4])


def test_branches(dev):
    b = Both(dev, pages=60, sequences=40, slots=5)
    b.reserve([21, 16, 0, 3], [0, 1, 2, 3])
    b.fork([0] * 12 + [1] * 3 + [2, 3, 3], list(range(4, 22)))
    b.fork([0, 0, 0], [30, 30, 31])                 # a child named twice
    b.fork([40, 0, KV_NONE, 0, 0], [32, 41, 33, KV_NONE, 34])
    b.fork([34, 4], [35, 36])                       # branches of branches
    b.fork([37, 0], [38, 37])                       # 37 is empty when 38 branches off
    b.free([0, 4, 34])
    b.fork([3] * 3, [0, 4, 34])
    b.compact()


def test_a_pool_too_small_for_the_branches(dev):
    b = Both(dev, pages=6, sequences=8, slots=5)
    b.reserve([12], [0])
    b.fork([0] * 6, [1, 2, 3, 4, 5, 6])             # four free pages for six copies
    b.free([1])
    b.fork([0], [6])


def test_a_trimmed_parent(dev):
    b = Both(dev, sequences=4, slots=8)
    b.reserve([50], [0])
    b.trim(10, 5)
    b.fork([0], [1])
    b.reserve([4, 4], [0, 1])
    b.trim(2, 0, [1, 1])
    b.free([0])
    b.compact()


@pytest.mark.parametrize("window,sinks", [(1, 0), (8, 0), (9, 1), (8, 8), (8, 9), (1000, 0),
                                          (1, 1 << 40), (1 << 40, 0), (24, 17)])
def test_trim(dev, window, sinks):
    b = Both(dev, sequences=5, pages=60, slots=12)
    b.reserve([0, 1, 8, 64, 95])
    b.trim(window, sinks)
    b.reserve([1] * 5)
    b.trim(window, sinks)


@pytest.mark.parametrize("pages,keep", [(1, 0.5), (63, 0.5), (64, 0.9), (1000, 0.3),
                                        (20000, 0.6), (20000, 0.0), (20000, 1.0)])
def test_large_pools(dev, pages, keep):
    """More pages than one step of the planning workgroup tests."""
    rng = np.random.default_rng(pages)
    seqs = 12
    slots = -(-pages // seqs) + 1
    b = Both(dev, layers=1, pages=pages, kv_heads=1, page=8, dim=8, sequences=seqs, slots=slots)
    b.reserve([min(pages // seqs, slots) * 8 + 1 if pages >= 2 * seqs else 1] * seqs)
    b.trim(8, 0, [s for s in range(seqs) if rng.random() > keep])
    b.free([s for s in range(seqs) if rng.random() > keep])
    b.compact()
    b.reserve([24] * seqs)


def test_many_sequences(dev):
    """More entries than the planning workgroup has lanes, in a mixed order."""
    rng = np.random.default_rng(3)
    b = Both(dev, layers=1, pages=9000, kv_heads=1, page=8, dim=8, sequences=3000, slots=4)
    order = rng.permutation(3000)
    b.reserve(rng.integers(0, 20, 3000), order)
    b.free(order[:1200])
    kids = [int(s) for s in order[:1200]]
    parents = [int(order[1200 + (i % 1500)]) for i in range(len(kids))]
    b.fork(parents, kids)
    b.compact()


def test_more_branches_than_a_workgroup_plans_at_once(dev):
    """Entries past the planning workgroup's lanes; a child that a later entry
    names as its parent counts as empty there; more marks and pages than LDS holds."""
    b = Both(dev, layers=1, pages=9000, kv_heads=1, page=8, dim=8, sequences=6000, slots=3)
    b.reserve([5, 17, 8], [0, 1, 2])
    kids = list(range(10, 2300))
    parents = [k % 3 for k in kids]
    parents[1500] = kids[3]
    b.fork(parents, kids)
    b.reserve([9] * 2400, list(range(2400)))
    b.free(kids[::2])
    b.compact()


@pytest.mark.parametrize("seed", range(6))
def test_random_lives(dev, seed):
    rng = np.random.default_rng(seed)
    n = int(rng.integers(2, 12))
    b = Both(dev, layers=int(rng.integers(1, 4)), pages=int(rng.integers(4, 60)),
             kv_heads=int(rng.integers(1, 4)), page=int(rng.choice([8, 16])),
             dim=int(rng.choice([8, 24, 64])), sequences=n, slots=int(rng.integers(1, 9)),
             dtype=[BF16, F16][seed & 1], seed=seed)
    for _ in range(12):
        seqs = [int(x) for x in rng.permutation(n)[:int(rng.integers(1, n + 1))]]
        what = rng.choice(["reserve", "reserve", "fork", "free", "trim", "compact"])
        if what == "reserve":
            b.reserve(rng.integers(0, 30, len(seqs)), seqs)
        elif what == "fork":
            b.fork([int(rng.integers(0, n)) for _ in seqs], seqs)
        elif what == "free":
            b.free(seqs)
        elif what == "trim":
            b.trim(int(rng.integers(1, 20)), int(rng.integers(0, 12)), seqs)
        else:
            b.compact()


def test_copy(dev):
    b = Both(dev, layers=3, dtype=F16)
    b.copy([3, 3, 7, 9], [1, 0, 39, 9])
    b.settle()
    b.copy([KV_NONE, 2, 5], [4, KV_NONE, 6])
    b.settle()
    b.m.copy([40, 2, 8], [4, 0xfffffff0, 11])
    b.dev.KVCopy(b.c, b.u32([40, 2, 8]), b.u32([4, 0xfffffff0, 11]))
    b.m.left_out = [0, 1]
    b.settle()


def test_pages_of_every_extent(dev):
    """Pages of 16 bytes a head to several strides of the copying workgroup."""
    for kv_heads, page, dim in [(1, 8, 8), (1, 8, 24), (3, 16, 40), (8, 16, 128), (5, 64, 256)]:
        b = Both(dev, pages=6, kv_heads=kv_heads, page=page, dim=dim)
        b.copy([0, 1], [4, 3])
        b.settle()
        b.reserve([page + 3] * 2, [0, 1])
        b.fork([0], [2])
        b.free([0])
        b.compact()


def narrow(x, dtype):
    """f32 to the cache's bits, nearest even (NaN stays one)."""
    import torch
    t = torch.from_numpy(np.ascontiguousarray(x, np.float32))
    t = t.to(torch.bfloat16 if dtype == BF16 else torch.float16)
    return t.view(torch.int16).numpy().view(np.uint16)


def rows(rng, shape, dtype):
    """Rows in a type: the values in f32 and the host array to upload."""
    x = (rng.standard_normal(shape) * np.exp2(rng.integers(-20, 12, shape))).astype(np.float32)
    x.flat[:6] = [0.0, -0.0, 65504.0, 1e-7, 2.0 ** -24, 1.00390625]
    if dtype == F32:
        return x, x
    bits = narrow(x, dtype)
    return (widen(bits, dtype)), bits


def widen(bits, dtype):
    if dtype == BF16:
        return (bits.astype(np.uint32) << 16).view(np.float32)
    return bits.view(np.float16).astype(np.float32)


@pytest.mark.parametrize("src", [F32, F16, BF16])
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_append(dev, src, dtype):
    rng = np.random.default_rng(7)
    b = Both(dev, dtype=dtype, kv_heads=3, dim=24)

    def put(layer, new, seqs=None, extra=0):
        n = len(new)
        off = np.concatenate([[0], np.cumsum(new)]).astype(np.uint32)
        k, kh = rows(rng, (int(off[-1]) + extra, 3, 24), src)
        v, vh = rows(rng, (int(off[-1]) + extra, 3, 24), src)
        with np.errstate(over="ignore"):
            kb, vb = narrow(k, dtype), narrow(v, dtype)
        one = all(x == 1 for x in new) and not extra
        b.m.append(layer, kb[:off[-1]], vb[:off[-1]], seqs, off)
        dev.KVAppend(b.c, layer, dev.upload(kh, src), dev.upload(vh, src), b.u32(seqs),
                     None if one else b.u32(off))
        assert n
        b.settle()

    b.reserve([9, 1, 16, 5, 0, 20])
    put(0, [9, 1, 16, 5, 0, 20])
    put(1, [1] * 3, [5, 2, 0])
    put(1, [3, 0, 17], [3, 4, 5], extra=6)           # rows past the last offset stay out
    put(0, [2, 3, 1], [0, KV_NONE, 2])               # a padded entry
    put(0, [2, 1], [1, 3])                           # more rows than the sequence holds
    put(0, [1, 1, 1], [6, 0, 0xfffffff0])            # outside the cache
    b.trim(4)
    put(1, [10, 2], [2, 0])                          # rows whose page was given back


def test_append_keeps_nan_and_infinities(dev):
    b = Both(dev, layers=1, kv_heads=1, dim=8, dtype=BF16)
    b.reserve([1], [0])
    x = np.array([np.nan, np.inf, -np.inf, 3.4e38, -3.4e38, 1e-40, 0, 1], np.float32)
    dev.KVAppend(b.c, 0, dev.upload(x.reshape(1, 1, 8)), dev.upload(x.reshape(1, 1, 8)),
                 b.u32([0]))
    dev.sync()
    page = b.m.tables[0, 0]
    got = widen(b.c.keys.numpy()[0, page, 0, 0], BF16)
    assert np.isnan(got[0]) and np.array_equal(got[1:], widen(narrow(x, BF16), BF16)[1:])


def test_pages_far_apart_in_a_large_cache(dev):
    """Element offsets past 32 bits: 2.2e9 elements a plane."""
    layers, pages, kv_heads, page, dim = 2, 2200, 8, 256, 256
    c = dev.kv_cache(layers, pages, kv_heads, page, dim, 2, pages)
    u = lambda x: dev.upload(np.asarray(x, np.uint32), U32)  # noqa: E731
    x = np.arange(kv_heads * dim, dtype=np.float32).reshape(1, kv_heads, dim) % 251
    # sequence 1 holds every page but the last; row 0 goes into the last one
    dev.KVReserve(c, u([(pages - 1) * page]), u([1]))
    dev.KVReserve(c, u([1]), u([0]))
    dev.KVAppend(c, 1, dev.upload(x), dev.upload(-x), u([0]))
    dev.KVFree(c, u([1]))
    dev.KVCompact(c)
    dev.sync()
    assert c.tables.numpy()[0, 0] == 0 and c.refs.numpy()[0] == 1
    elems = kv_heads * page * dim
    # page 0 of layer 1, where the compaction moved it
    host = np.empty((kv_heads, page, dim), np.uint16)
    for plane, want in ((c.keys, x), (c.values, -x)):
        accel_amd._check(accel_amd.lib().accel_hip_read(
            dev.index, plane.ptr, pages * elems * 2, host.ctypes.data, host.nbytes))
        assert np.array_equal(widen(host[:, 0], BF16), want[0])
    c.free()


def test_the_calls_replay_in_a_graph(dev):
    """reserve and append captured once, replayed as a decode loop runs them."""
    st = dev.stream()
    b = Both(dev, layers=1, kv_heads=1, dim=8, sequences=3, pages=30)
    grow, seqs = b.u32([1, 3, 1]), b.u32([2, 0, KV_NONE])
    off = b.u32([0, 1, 4, 5])
    k, kh = rows(np.random.default_rng(1), (5, 1, 8), F32)
    kb = dev.upload(kh)

    def step():
        dev.KVReserve(b.c, grow, seqs, st)
        dev.KVAppend(b.c, 0, kb, kb, seqs, off, st)

    def model():
        b.m.reserve([1, 3, 1], [2, 0, KV_NONE])
        n = narrow(k, BF16)
        b.m.append(0, n, n, [2, 0, KV_NONE], [0, 1, 4, 5])

    step()
    dev.sync(st)
    model()
    b.check()
    dev.capture_begin(st)
    step()
    ex = dev.capture_end(st)
    for _ in range(4):
        dev.launch(ex, st)
        dev.sync(st)
        model()
        b.check()
        b.reserve([2], [1])               # eager work between the replays
    dev.destroy_exec(ex)
    dev.destroy_stream(st)
