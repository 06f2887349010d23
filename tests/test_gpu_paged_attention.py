"""PagedAttention and PagedPrefill on the GPU against attention in 64 bits from
its definition (oracle/kvcache_np.py).

The bound, per output element, from the operations' roundings (u = 2^-24 the
f32 half step, S the row's largest sum of |q k| * scale plus its spread of
scores, M = sum w |v|):
- a score is a sum of dim products and a scaling: at most (dim + 4) u S off, and
  the exponential's argument and result add 4 u S + 4 u, so a weight is off by
  d = (dim + 8) u S + 4 u of itself, and the quotient by at most 2 d M;
- sums over n keys run in chains of at most n / 16 + 64 additions and joins:
  twice that (the values' sum and the weights') times u M;
- queries and weights of f32 calls are split into terms that hold 2^-22 of
  them at least: 2^-21 (S + 1) M more;
- prompts in a 16-bit type round each weight to it: half a step of it, M;
- the result is rounded once to its type: half a step of the value.
"""
import numpy as np
import pytest

import accel_amd
from accel_amd import BF16, F16, F32, U32, KV_NONE
from oracle import kvcache_np
from test_gpu_kv_pages import narrow, widen

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
HALF = {F32: 2.0 ** -24, F16: 2.0 ** -11, BF16: 2.0 ** -8}


def bound(want, mass, size, q_dtype, dtype, dim, n, prompt):
    S = size[..., None]
    d = (dim + 8) * U * S + 4 * U
    err = (2 * d + 2 * (n / 16 + 64) * U) * mass
    if q_dtype == F32:
        err = err + 2.0 ** -21 * (S + 1) * mass
    elif prompt:
        err = err + HALF[dtype] * mass
    # f16 results below the normal range are rounded to steps of 2^-24
    return err + HALF[q_dtype] * np.abs(want) + (2.0 ** -25 if q_dtype == F16 else 1e-37)


def as_type(x, t):
    """Values as a type holds them, and the array to upload."""
    if t == F32:
        x = x.astype(np.float32)
        return x, x
    bits = narrow(x, t)
    return widen(bits, t), bits


class Case:
    """A cache of `lens` tokens in shuffled pages, and queries."""

    def __init__(self, dev, lens, new=None, heads=4, kv_heads=2, dim=64, page=16, q=BF16, kv=BF16,
                 layers=1, seqs=None, seed=0, gain=2.0, extra_rows=0, kv_gain=1.0):
        rng = np.random.default_rng(seed)
        self.dev, self.dim, self.q_dtype, self.kv = dev, dim, q, kv
        self.heads, self.layers = heads, layers
        slots = max(1, -(-max(lens, default=1) // page) + 1)
        need = [-(-n // page) for n in lens]
        pages = sum(need) + 3
        order = rng.permutation(pages)
        self.tables = np.full((len(lens), slots), KV_NONE, np.uint32)
        at = 0
        for i, n in enumerate(need):
            self.tables[i, :n] = order[at:at + n]
            at += n
        self.lens = np.asarray(lens, np.uint32)
        shape = (layers, pages, kv_heads, page, dim)
        self.k, self.kh = as_type(rng.standard_normal(shape) * kv_gain, kv)
        self.v, self.vh = as_type(rng.standard_normal(shape) * kv_gain, kv)
        # what no position holds is never read as one
        held = np.zeros((pages, page), bool)
        for i, n in enumerate(lens):
            for p in range(n):
                held[self.tables[i, p // page], p % page] = True
        nan = 0x7fc0 if kv == BF16 else 0x7e00
        for bits in (self.kh, self.vh):
            np.moveaxis(bits, 2, 3)[:, ~held] = nan
        self.seqs = np.arange(len(lens)) if seqs is None else np.asarray(seqs)
        self.listed = seqs is not None
        self.new = None if new is None else list(new)
        counts = [1] * len(self.seqs) if new is None else self.new
        self.off = np.concatenate([[0], np.cumsum(counts)]).astype(np.uint32)
        T = int(self.off[-1]) + extra_rows
        self.q, self.qh = as_type(rng.standard_normal((T, heads, dim)) * gain, q)
        self.T = T
        self.left_out = False

    def upload(self):
        d = self.dev
        u = lambda x: d.upload(np.ascontiguousarray(x, np.uint32), U32)  # noqa: E731
        kv = d.upload(self.kh, self.kv), d.upload(self.vh, self.kv)
        refs = np.zeros(self.k.shape[1], np.uint32)
        self.cache = accel_amd.KVCache(d, *kv, u(refs), u(self.tables), u(self.lens))
        self.qb = d.upload(self.qh, self.q_dtype)
        # rows that no entry covers have to stay what they were
        self.fill = np.full(self.qh.shape, 7 if self.q_dtype == F32 else 0x4321, self.qh.dtype)
        self.out = d.upload(self.fill, self.q_dtype)
        self.seqs_b = u(self.seqs) if self.listed else None
        self.off_b = u(self.off)

    def call(self, layer=0, scale=0.0, window=0, sinks=0, stream=None):
        kw = dict(layer=layer, seqs=self.seqs_b, scale=scale, window=window, sinks=sinks,
                  stream=stream)
        if self.new is None:
            self.dev.PagedAttention(self.qb, self.cache, self.out, **kw)
        else:
            self.dev.PagedPrefill(self.qb, self.off_b, self.cache, self.out, **kw)

    def got(self):
        bits = self.out.numpy()
        return bits if self.q_dtype == F32 else widen(bits, self.q_dtype)

    def want(self, layer=0, scale=0.0, window=0, sinks=0):
        scale = scale or float(np.float32(self.dim ** -0.5))
        return kvcache_np.attention(self.q.astype(np.float64), self.k[layer].astype(np.float64),
                                    self.v[layer].astype(np.float64), self.tables, self.lens,
                                    self.seqs, self.off, scale, window, sinks)

    def compare(self, **kw):
        want, mass, size = self.want(**kw)
        got = self.got().astype(np.float64)
        n = int(self.off[-1])
        tol = bound(want, mass, size, self.q_dtype, self.kv, self.dim, int(max(self.lens, default=0)),
                    self.new is not None)
        bad = ~(np.abs(got - want) <= tol)
        bad[n:] = False
        assert not bad.any(), (np.argwhere(bad)[:5], got[bad][:5], want[bad][:5], tol[bad][:5])
        # nothing seen: exactly zero; rows past the last offset: untouched
        assert not got[:n][(mass[:n] == 0) & (want[:n] == 0)].any()
        bits = self.out.numpy()
        assert np.array_equal(bits[n:], self.fill[n:])

    def check(self, **kw):
        self.upload()
        self.call(**kw)
        if self.left_out:
            with pytest.raises(accel_amd.AccelError, match="left out"):
                self.dev.sync()
        self.dev.sync()
        self.compare(**kw)
        self.free()

    def free(self):
        self.cache.free()
        for b in (self.qb, self.out, self.off_b, self.seqs_b):
            if b is not None:
                b.free()


TYPES = [(F32, BF16), (F32, F16), (BF16, BF16), (F16, F16)]
ids = {F32: "f32", F16: "f16", BF16: "bf16"}
types = pytest.mark.parametrize("q,kv", TYPES, ids=[f"{ids[a]}-{ids[b]}" for a, b in TYPES])


# ---- one new token -------------------------------------------------------------

@types
@pytest.mark.parametrize("n", [0, 1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 300])
def test_decode_lengths(dev, q, kv, n):
    Case(dev, [n], q=q, kv=kv, seed=n).check()


@types
@pytest.mark.parametrize("dim", [8, 16, 24, 40, 64, 72, 80, 96, 120, 128, 136, 192, 248, 256])
def test_decode_head_dims(dev, q, kv, dim):
    Case(dev, [70, 3, 41], dim=dim, q=q, kv=kv, seed=dim).check()


@types
@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (3, 1), (4, 4), (6, 3), (8, 1), (14, 2),
                                            (16, 1), (17, 1), (40, 1), (96, 2), (32, 8)])
def test_decode_groups(dev, q, kv, heads, kv_heads):
    Case(dev, [45, 100], heads=heads, kv_heads=kv_heads, q=q, kv=kv, seed=heads).check()


@pytest.mark.parametrize("page", [8, 16, 32, 64, 128, 512, 4096])
def test_decode_pages(dev, page):
    Case(dev, [1, page - 1, page, page + 1, 2 * page + 7], page=page, seed=page).check()


@types
def test_decode_ragged_batch(dev, q, kv):
    rng = np.random.default_rng(5)
    lens = [int(x) for x in np.exp(rng.uniform(0, np.log(1500), 40))] + [0, 0, 1]
    Case(dev, lens, heads=4, kv_heads=1, q=q, kv=kv).check()


@types
@pytest.mark.parametrize("dim", [40, 64, 128, 200])
@pytest.mark.parametrize("n", [61, 150])
def test_decode_many_short_sequences(dev, q, kv, dim, n):
    """Enough sequences that runs of short ones go to a wave each, long and
    empty ones between them; a lane's or a table's lookup of them."""
    rng = np.random.default_rng(n)
    lens = [int(x) for x in rng.integers(0, 200, n)]
    for i in (5, 17, 18, 40):
        lens[i] = 0
    lens[11], lens[30], lens[-1] = 900, 390, 1
    seqs = [int(x) for x in rng.permutation(n)]
    seqs[7] = KV_NONE
    # heads of one group each: 512 pairs or more
    heads = -(-512 // n)
    Case(dev, lens, heads=heads, kv_heads=heads, dim=dim, page=8, q=q, kv=kv, seqs=seqs,
         seed=n).check()
    Case(dev, lens, heads=heads, kv_heads=heads, dim=dim, page=8, q=q, kv=kv, seqs=seqs,
         seed=n).check(window=70, sinks=5)


@types
@pytest.mark.parametrize("n", [4000, 20001])
def test_decode_split_over_a_long_cache(dev, q, kv, n):
    Case(dev, [n, 5, n // 3], heads=2, kv_heads=1, q=q, kv=kv, seed=n).check()


@types
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (16, 0), (17, 4), (64, 4), (100, 33),
                                          (5, 200), (10000, 3), (1 << 40, 7)])
def test_decode_window_and_sinks(dev, q, kv, window, sinks):
    Case(dev, [0, 1, 16, 17, 30, 64, 200, 333], q=q, kv=kv).check(window=window, sinks=sinks)


def test_decode_window_over_pages_given_back(dev):
    c = Case(dev, [400, 90, 1300], page=16)
    for i, n in enumerate([400, 90, 1300]):
        for j in range(c.tables.shape[1]):
            if j * 16 >= 5 and (j + 1) * 16 <= n - 50:
                c.tables[i, j] = KV_NONE
    c.check(window=50, sinks=5)


def test_decode_lists_padding_and_the_same_sequence_twice(dev):
    Case(dev, [40, 7, 100, 0], seqs=[2, KV_NONE, 0, 0, 3, KV_NONE, 1, 2]).check()


def test_decode_layers_and_scale(dev):
    c = Case(dev, [40, 70], layers=3)
    for layer in range(3):
        c.check(layer=layer, scale=0.05 * (layer + 1))


def test_decode_bad_pages_and_sequences_are_left_out(dev):
    c = Case(dev, [100, 100, 64], seqs=[0, 1, 9, 2])
    c.tables[0, 2] = 0x7fffffff
    c.tables[1, :] = KV_NONE
    c.left_out = True
    c.check()


def test_decode_length_past_its_table(dev):
    # a length past what the slots hold counts as what they hold
    c = Case(dev, [64])
    c.lens[0] = 80                       # five slots of 16: the last has no page
    c.left_out = True
    c.check()
    c.lens[0] = 0xffffffff
    c.upload()
    c.call()
    with pytest.raises(accel_amd.AccelError, match="left out"):
        c.dev.sync()
    c.lens[0] = 80
    c.compare()
    c.free()


@types
def test_decode_extreme_scores(dev, q, kv):
    """Scores hundreds apart (one key has all the weight), equal scores, and
    values near the type's ends."""
    Case(dev, [200, 33], q=q, kv=kv, gain=60.0).check()
    c = Case(dev, [200, 33], q=q, kv=kv)
    c.q[:], c.qh[:] = 0, 0
    c.check()
    Case(dev, [200, 33], q=q, kv=kv, gain=1e-4, kv_gain=1e-3).check()
    Case(dev, [200, 33], q=q, kv=kv, gain=1e-3, kv_gain=2e3).check()


def test_decode_nan_and_infinities_where_they_are_seen_or_not(dev):
    for bits in (0x7f80, 0xff80, 0x7fc0):
        c = Case(dev, [200, 150], heads=4, kv_heads=2)
        # position 10 is outside both windows; its keys and values are anything
        for i in range(2):
            c.kh[0, c.tables[i, 0], :, 10] = bits
            c.vh[0, c.tables[i, 0], :, 10] = bits
            # and position 149 of sequence 1 is seen by it: not finite there
        c.vh[0, c.tables[1, 149 // 16], 0, 149 % 16, 5] = bits
        c.upload()
        c.call(window=60, sinks=4)
        c.dev.sync()
        got = c.got()
        assert not np.isfinite(got[1, :2, 5]).any()
        want, mass, size = c.want(window=60, sinks=4)
        got[1, :2, 5] = want[1, :2, 5]
        tol = bound(want, mass, size, BF16, BF16, 64, 200, False)
        assert (np.abs(got - want) <= tol).all()
        c.free()


def test_decode_repeats_itself(dev):
    """The join of a split cache adds in a fixed order."""
    c = Case(dev, [9000, 100, 4000], heads=8, kv_heads=2, dim=128, q=F32)
    c.upload()
    first = None
    for _ in range(5):
        c.call()
        c.dev.sync()
        got = c.out.numpy()
        assert first is None or np.array_equal(first, got)
        first = got
    c.compare()
    c.free()


# ---- prompts --------------------------------------------------------------------

@types
@pytest.mark.parametrize("n", [1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 200])
def test_prompt_lengths(dev, q, kv, n):
    Case(dev, [n], new=[n], q=q, kv=kv, seed=n).check()


@types
@pytest.mark.parametrize("dim", [8, 24, 64, 80, 96, 120, 128, 136, 192, 256])
def test_prompt_head_dims(dev, q, kv, dim):
    Case(dev, [70, 41], new=[70, 13], dim=dim, q=q, kv=kv, seed=dim).check()


@types
@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (3, 1), (4, 4), (6, 3), (7, 1), (16, 1),
                                            (17, 1), (40, 1), (32, 8)])
def test_prompt_groups(dev, q, kv, heads, kv_heads):
    Case(dev, [45, 90], new=[45, 33], heads=heads, kv_heads=kv_heads, q=q, kv=kv,
         seed=heads).check()


@pytest.mark.parametrize("page", [8, 16, 32, 64, 128, 4096])
def test_prompt_pages(dev, page):
    Case(dev, [page + 1, 2 * page, 40], new=[min(page + 1, 70), 9, 40], page=page,
         seed=page).check()


@types
def test_prompt_chunks_after_prefixes(dev, q, kv):
    Case(dev, [500, 64, 7, 333, 900, 130], new=[1, 64, 7, 100, 3, 65], q=q, kv=kv,
         heads=6, kv_heads=2).check()


@types
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (16, 0), (17, 4), (64, 4), (100, 33),
                                          (5, 200), (10000, 3)])
def test_prompt_window_and_sinks(dev, q, kv, window, sinks):
    Case(dev, [230, 64, 300], new=[230, 20, 77], q=q, kv=kv).check(window=window, sinks=sinks)


def test_prompt_window_over_pages_given_back(dev):
    c = Case(dev, [700, 300], new=[100, 40], page=16)
    for i, (n, new) in enumerate([(700, 100), (300, 40)]):
        for j in range(c.tables.shape[1]):
            if j * 16 >= 5 and (j + 1) * 16 <= n - new - 50 + 1:
                c.tables[i, j] = KV_NONE
    c.check(window=50, sinks=5)


def test_prompt_padding_empty_entries_and_rows_behind(dev):
    Case(dev, [40, 7, 100, 30], new=[40, 5, 0, 64, 0, 9], seqs=[0, KV_NONE, 1, 2, 3, 3],
         extra_rows=21).check()


def test_prompt_more_rows_than_positions(dev):
    # rows before a sequence's first position see nothing
    Case(dev, [5, 0, 70], new=[20, 4, 70]).check()


@types
def test_prompt_one_row_an_entry(dev, q, kv):
    Case(dev, [100, 1, 0, 63], new=[1, 1, 1, 1], q=q, kv=kv).check()


def test_prompt_many_entries(dev):
    rng = np.random.default_rng(9)
    new = [int(x) for x in rng.integers(0, 12, 300)]
    Case(dev, [int(n + x) for n, x in zip(new, rng.integers(0, 40, 300))], new=new, heads=2,
         kv_heads=1, dim=16, page=8).check()


def test_prompt_layers_and_scale(dev):
    c = Case(dev, [90, 70], new=[90, 11], layers=3)
    for layer in range(3):
        c.check(layer=layer, scale=0.05 * (layer + 1))


def test_prompt_bad_pages_and_sequences_are_left_out(dev):
    c = Case(dev, [100, 100, 64], new=[50, 20, 9, 64], seqs=[0, 1, 9, 2])
    c.tables[0, 2] = 0x7fffffff
    c.tables[1, :] = KV_NONE
    c.left_out = True
    c.check()


@types
def test_prompt_extreme_scores(dev, q, kv):
    Case(dev, [140], new=[140], q=q, kv=kv, gain=60.0).check()
    c = Case(dev, [140], new=[140], q=q, kv=kv)
    c.q[:], c.qh[:] = 0, 0
    c.check()
    Case(dev, [140], new=[140], q=q, kv=kv, gain=1e-4, kv_gain=1e-3).check()
    Case(dev, [140], new=[140], q=q, kv=kv, gain=1e-3, kv_gain=2e3).check()


@types
@pytest.mark.parametrize("bits", ["inf", "-inf", "nan"])
def test_prompt_values_that_are_not_finite_reach_only_who_sees_them(dev, q, kv, bits):
    """A key and a value late in the prompt are not finite: the queries before
    them, and those whose window has passed them, are what they were."""
    x = {"inf": np.inf, "-inf": -np.inf, "nan": np.nan}[bits]
    b = narrow(np.array([x], np.float32), kv)[0]
    for window, sinks in ((0, 0), (40, 3)):
        c = Case(dev, [150], new=[120], q=q, kv=kv, heads=4, kv_heads=2, dim=64)
        where = c.tables[0, 77 // 16], 77 % 16
        c.vh[0, where[0], :, where[1], 3:60:7] = b
        c.kh[0, c.tables[0, 101 // 16], :, 101 % 16, 9] = b
        c.upload()
        c.call(window=window, sinks=sinks)
        c.dev.sync()
        got = c.got()
        want, mass, size = c.want(window=window, sinks=sinks)
        tol = bound(want, mass, size, q, kv, 64, 150, True)
        p = np.arange(30, 150)
        sees = lambda j: (p >= j) & ((p - j < window) | (window == 0))  # noqa: E731
        clean = ~sees(77) & ~sees(101)
        assert clean.sum() >= 40
        assert (np.abs(got - want) <= tol)[clean].all()
        # a value that is seen shows, in its own columns alone
        value = sees(77) & ~sees(101)
        cols = np.zeros(64, bool)
        cols[3:60:7] = True
        assert not np.isfinite(got[value][..., cols]).any()
        assert (np.abs(got - want) <= tol)[value][..., ~cols].all()
        if bits == "nan":
            assert np.isnan(got[sees(101)]).all()
        c.free()


@types
@pytest.mark.parametrize("window,sinks", [(0, 0), (1500, 30)])
def test_prompt_few_rows_after_a_long_prefix(dev, q, kv, window, sinks):
    """Tiles of rows that several workgroups share, joined in a fixed order."""
    c = Case(dev, [3000, 700, 2100, 0], new=[5, 64, 1, 0], heads=4, kv_heads=2, q=q, kv=kv)
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


def test_prompt_few_rows_heads_of_256(dev):
    Case(dev, [1500, 900], new=[7, 40], heads=6, kv_heads=2, dim=256).check()
    Case(dev, [1500, 900], new=[7, 40], heads=6, kv_heads=2, dim=200, q=F32).check()


def test_a_long_prompt_in_blocks(dev):
    """Rows of a prompt of several tiles against the same prompt in chunks."""
    n = 1100
    c = Case(dev, [n], new=[n], heads=8, kv_heads=2, dim=128, q=F32)
    c.upload()
    c.call(window=400, sinks=2)
    dev.sync()
    whole = c.out.numpy()
    for a, b in [(0, 300), (300, 301), (301, 1100)]:
        d = Case(dev, [n], new=[b - a], heads=8, kv_heads=2, dim=128, q=F32)
        d.k, d.v, d.kh, d.vh, d.tables = c.k, c.v, c.kh, c.vh, c.tables
        d.q, d.qh = c.q[a:b].copy(), c.qh[a:b].copy()
        d.lens[0] = b
        d.upload()
        d.call(window=400, sinks=2)
        dev.sync()
        # f32 calls: two results within the bounds' sum of each other; a 64-bit
        # oracle of the whole would take long here
        assert np.abs(d.out.numpy() - whole[a:b]).max() <= 2e-4
        d.free()
    c.free()


def test_keys_far_apart_in_a_large_cache(dev):
    """Offsets past 32 bits: the last pages of layer 1 of 2.3e9 elements a plane
    give what the first pages of a small cache give, bit for bit."""
    rng = np.random.default_rng(2)
    KV, P, D, H, n = 8, 256, 256, 16, 700
    k, v = (rng.standard_normal((n, KV, D)).astype(np.float32) for _ in range(2))
    q = narrow(rng.standard_normal((40, H, D)) * 2, BF16)
    u = lambda x: dev.upload(np.asarray(x, np.uint32), U32)  # noqa: E731
    res = []
    for layers, pages, before in ((2, 2200, 2197), (1, 3, 0)):
        c = dev.kv_cache(layers, pages, KV, P, D, 2, 2200)
        if before:
            dev.KVReserve(c, u([before * P]), u([1]))
        dev.KVReserve(c, u([n]), u([0]))
        dev.KVAppend(c, layers - 1, dev.upload(k), dev.upload(v), u([0]), u([0, n]))
        one, many = dev.alloc((1, H, D), BF16), dev.alloc((40, H, D), BF16)
        dev.PagedAttention(dev.upload(q[:1], BF16), c, one, layer=layers - 1, seqs=u([0]))
        dev.PagedPrefill(dev.upload(q, BF16), u([0, 40]), c, many, layer=layers - 1, seqs=u([0]))
        dev.sync()
        assert c.tables.numpy()[0, 0] == before
        res.append((one.numpy(), many.numpy()))
        c.free()
    for a, b in zip(*res):
        assert np.array_equal(a, b) and np.isfinite(widen(a, BF16)).all()


# ---- together ---------------------------------------------------------------------

@types
def test_a_generation(dev, q, kv):
    """Prompts in two chunks, then tokens: pages reserved, rows appended,
    attention over them, a branch that goes its own way, a page given back and
    a compaction, as a serving loop does, against all of it restated."""
    rng = np.random.default_rng(11)
    L, KV, H, D, P = 2, 2, 6, 40, 8
    c = dev.kv_cache(L, 60, KV, P, D, 4, 20, kv)
    m = kvcache_np.Pages(np.zeros((L, 60, KV, P, D), np.float32),
                         np.zeros((L, 60, KV, P, D), np.float32), 4, 20)
    u = lambda x: dev.upload(np.asarray(x, np.uint32), U32)  # noqa: E731

    def step(seqs, new, one=False, window=0, sinks=0):
        off = np.concatenate([[0], np.cumsum(new)]).astype(np.uint32)
        T = int(off[-1])
        m.reserve(new, seqs)
        dev.KVReserve(c, u(new), u(seqs))
        for layer in range(L):
            qv, qh = as_type(rng.standard_normal((T, H, D)) * 2, q)
            kr = rng.standard_normal((T, KV, D)).astype(np.float32)
            vr = rng.standard_normal((T, KV, D)).astype(np.float32)
            m.append(layer, widen(narrow(kr, kv), kv), widen(narrow(vr, kv), kv), seqs, off)
            dev.KVAppend(c, layer, dev.upload(kr), dev.upload(vr), u(seqs), None if one else u(off))
            out = dev.alloc((T, H, D), q)
            if one:
                dev.PagedAttention(dev.upload(qh, q), c, out, layer=layer, seqs=u(seqs),
                                   window=window, sinks=sinks)
            else:
                dev.PagedPrefill(dev.upload(qh, q), u(off), c, out, layer=layer, seqs=u(seqs),
                                 window=window, sinks=sinks)
            dev.sync()
            got = out.numpy() if q == F32 else widen(out.numpy(), q)
            want, mass, size = kvcache_np.attention(
                qv.astype(np.float64), m.keys[layer].astype(np.float64),
                m.values[layer].astype(np.float64), m.tables, m.lens, seqs, off,
                float(np.float32(D ** -0.5)), window, sinks)
            tol = bound(want, mass, size, q, kv, D, int(m.lens.max()), not one)
            assert (np.abs(got - want) <= tol).all()

    step([2, 0], [30, 11])
    step([2, 0], [5, 20])
    step([0, 2], [1, 1], one=True)
    m.fork([2, 2], [1, 3])
    dev.KVFork(c, u([2, 2]), u([1, 3]))
    for _ in range(9):
        step([3, 1, 2, 0], [1, 1, 1, 1], one=True)
    m.trim(12, 2, [2, 0])
    dev.KVTrim(c, 12, 2, u([2, 0]))
    step([0, 2], [1, 1], one=True, window=12, sinks=2)
    m.free([3])
    dev.KVFree(c, u([3]))
    m.compact()
    dev.KVCompact(c)
    step([1, 0], [1, 1], one=True, window=12, sinks=2)
    step([1, 2], [10, 3], window=12, sinks=2)
    for name in ("refs", "tables", "lens"):
        assert np.array_equal(getattr(c, name).numpy(), getattr(m, name)), name
    c.free()


@pytest.mark.parametrize("prompt", [False, True])
def test_replays_and_streams(dev, prompt):
    """Captured once on a stream of its own and replayed, lengths changing
    between the replays, beside another captured call on the same workspace."""
    st = dev.stream()
    a = Case(dev, [3000, 500], new=[3, 70] if prompt else None, heads=8, kv_heads=2, dim=128,
             q=F32)
    b = Case(dev, [900], new=[40] if prompt else None, heads=4, kv_heads=1, seed=3)
    execs = []
    for c in (a, b):
        c.upload()
        c.call(stream=st)
        dev.sync(st)
        c.compare()
        dev.capture_begin(st)
        c.call(stream=st)
        execs.append(dev.capture_end(st))
    for n in (2999, 100, 1, 3000):
        a.lens[0] = n
        a.cache.lens.write(a.lens)
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
