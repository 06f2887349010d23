"""The paged cache and its attention at the edges of what the header allows:
arguments near their types' ends, values that are not finite, queries and
scales that leave the normal range, weights far below the largest, a pool that
runs short.  Bounds are those of test_gpu_paged_attention.py unless said."""
import numpy as np
import pytest

import accel_amd
from accel_amd import BF16, F16, F32, U32, KV_NONE
from test_gpu_kv_pages import Both, narrow
from test_gpu_paged_attention import Case, bound, types

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("window,sinks", [(1, 2 ** 63 - 1), (8, 2 ** 63 - 8), (1, 2 ** 31),
                                          (2 ** 63 - 1, 0), (2 ** 63 - 1, 2 ** 63 - 1)])
def test_trim_with_windows_and_sinks_past_any_table(dev, window, sinks):
    b = Both(dev, sequences=5, pages=60, slots=12)
    b.reserve([0, 1, 8, 64, 95])
    b.trim(window, sinks)
    assert (b.m.tables != KV_NONE).sum() == 22       # nothing is given back


# ---- more work than one launch's lanes, which are counted in 32 bits ------------

MANY = (1 << 24) + 9


def test_more_sequences_than_a_launch_has_blocks(dev):
    """Pages given back by lists, and by all sequences, past 2^24 of them."""
    c = dev.kv_cache(1, 8, 1, 8, 8, MANY, 2)
    u = lambda x: dev.upload(np.asarray(x, np.uint32), U32)  # noqa: E731
    some = [0, MANY // 2, MANY - 1]
    order = dev.upload(np.arange(MANY, dtype=np.uint32)[::-1].copy(), U32)
    dev.KVReserve(c, u([16, 16, 16]), u(some))
    dev.KVTrim(c, 8)
    dev.sync()
    t = c.tables.numpy()
    assert (t[some, 0] == KV_NONE).all() and (t[some, 1] != KV_NONE).all()
    assert c.refs.numpy().sum() == 3
    dev.KVFree(c, order)
    dev.KVReserve(c, u([16, 16, 16]), u(some))
    dev.sync()
    assert (c.tables.numpy()[some] == np.arange(6).reshape(3, 2)).all()
    dev.KVFree(c)
    dev.sync()
    assert not c.refs.numpy().any() and not c.lens.numpy().any()
    assert (c.tables.numpy() == KV_NONE).all()
    c.free()


def test_more_copies_and_branches_than_a_launch_has_blocks(dev):
    """2 blocks a pair and 3 a branch, all but the first and last are padding."""
    b = Both(dev, layers=1, pages=12, sequences=5, slots=4)
    b.reserve([11, 20], [0, 1])
    n = MANY // 2 + 1

    def padded(first, last):
        x = np.full(n, KV_NONE, np.uint32)
        x[0], x[-1] = first, last
        return dev.upload(x, U32)

    b.m.copy([0, 1], [9, 11])
    dev.KVCopy(b.c, padded(0, 1), padded(9, 11))
    b.settle()
    b.m.fork([0, 1], [2, 3])
    dev.KVFork(b.c, padded(0, 1), padded(2, 3))
    b.settle()


def test_more_rows_than_a_launch_has_lanes(dev):
    """2^32 and some pieces of rows of which the last row alone has a sequence
    (64 GB of rows, not read)."""
    T, KV, D = 32769, 4096, 256
    c = dev.kv_cache(1, 2, KV, 8, D, 1, 2)
    u = lambda x: dev.upload(np.asarray(x, np.uint32), U32)  # noqa: E731
    rows = dev.alloc((T, KV, D), BF16)
    last = np.random.default_rng(4).integers(0, 1 << 16, (KV, D)).astype(np.uint16)
    accel_amd._check(accel_amd.lib().accel_hip_write(
        dev.index, rows.ptr, (T - 1) * KV * D * 2, last.ctypes.data, last.nbytes))
    dev.KVReserve(c, u([11]))
    dev.KVAppend(c, 0, rows, rows, u([KV_NONE, 0]), u([0, T - 1, T]))
    dev.sync()
    for plane in (c.keys, c.values):
        assert np.array_equal(plane.numpy()[0, 1, :, 2], last)
    rows.free()
    c.free()


def test_more_prompt_tiles_than_a_launch_has_blocks(dev):
    """Entries of a token each, 2^24 tiles of rows and some: each of them as in
    a short list."""
    n, period = 2_100_000, 5
    c = Case(dev, [40, 7, 100, 0, 63], new=[1] * period, heads=8, kv_heads=8, dim=8, page=8)
    c.upload()
    c.call()
    dev.sync()
    c.compare()
    want = c.out.numpy()
    q = dev.upload(np.tile(c.qh, (n // period, 1, 1)), BF16)
    out = dev.alloc((n, 8, 8), BF16)
    dev.PagedPrefill(q, dev.upload(np.arange(n + 1, dtype=np.uint32), U32), c.cache, out,
                     seqs=dev.upload(np.arange(n, dtype=np.uint32) % period, U32))
    dev.sync()
    got = out.numpy().reshape(n // period, *want.shape)
    assert (got == want).all()
    c.free()


def test_rows_of_an_entry_past_half_of_31_bits(dev):
    """2^30 empty entries before the one that has a row: places in the offsets
    whose sum passes 31 bits."""
    n = (1 << 30) + 5
    c = dev.kv_cache(1, 2, 1, 8, 8, n, 1)
    lib = accel_amd.lib()

    def put(buffer, at, x):
        x = np.asarray(x, np.uint32)
        accel_amd._check(lib.accel_hip_write(dev.index, buffer.ptr, 4 * at, x.ctypes.data,
                                             x.nbytes))

    put(c.lens, n - 1, [1])
    put(c.tables, n - 1, [1])
    off = dev.alloc((n + 1,), U32)
    zeros = np.zeros(1 << 26, np.uint32)
    for at in range(0, n, len(zeros)):
        put(off, at, zeros[:n - at])
    put(off, n, [1])
    x = np.arange(8, dtype=np.uint16).reshape(1, 1, 8)
    row = dev.upload(x, BF16)
    dev.KVAppend(c, 0, row, row, None, off)
    dev.sync()
    assert np.array_equal(c.keys.numpy()[0, 1, 0, 0], x[0, 0])
    off.free()
    c.free()


@types
@pytest.mark.parametrize("prompt", [False, True])
@pytest.mark.parametrize("scale", [1e-45, 1e-41, 2e-38])
def test_scales_below_the_normal_range(dev, q, kv, prompt, scale):
    """All scores are nearly 0 and all weights nearly equal; keys that a row
    does not see stay out of it."""
    Case(dev, [140, 70], new=[140, 9] if prompt else None, q=q, kv=kv).check(scale=scale)
    Case(dev, [140, 70], new=[140, 9] if prompt else None, q=q, kv=kv).check(
        scale=scale, window=20, sinks=3)


@pytest.mark.parametrize("kv", [F16, BF16])
@pytest.mark.parametrize("prompt", [False, True])
def test_f32_queries_below_the_normal_range(dev, kv, prompt):
    """Rows whose largest element is anything down to the smallest subnormal,
    beside ordinary rows; under the usual scale, and one that lifts them."""
    rng = np.random.default_rng(5)
    for scale in (0.0, 1e30):
        c = Case(dev, [140, 70], new=[140, 9] if prompt else None, q=F32, kv=kv, kv_gain=0.01)
        size = 2.0 ** rng.integers(-149, -100, c.q.shape[:2])
        size[::3] = 2.0 ** -149
        if not scale:
            size[1::3] = 1
        x = (rng.standard_normal(c.q.shape) * size[..., None]).astype(np.float32)
        c.q[:], c.qh[:] = x, x
        c.check(scale=scale)
        c.check(scale=scale, window=20, sinks=3)


def seen_not_finite(dev, q, kv, new, lens, put_k=(), put_v=(), tiny=(), **kw):
    """A case with keys' or values' elements set to what is not finite, run and
    compared: (sequence, position, head, dim, value) each.  The result has to be
    what 64 bits give, infinities and NaN where they are; elsewhere within the
    bounds, the scores' part of them from the keys without those elements."""
    c = Case(dev, lens, new=new, heads=4, kv_heads=2, dim=64, q=q, kv=kv, seed=17, **kw)
    for row, dim, x in tiny:
        c.q[row, :, dim] = c.qh[row, :, dim] = x
    _, _, size = c.want()
    for bits, held, puts in ((c.kh, c.k, put_k), (c.vh, c.v, put_v)):
        for s, pos, h, d, x in puts:
            at = 0, c.tables[s, pos // 16], h, pos % 16, d
            held[at] = x
            bits[at] = narrow(np.array([x], np.float32), kv)[0]
    with np.errstate(invalid="ignore"):
        want, _, _ = c.want()
        c.v = np.nan_to_num(c.v, nan=0.0, posinf=0.0, neginf=0.0)
        _, mass, _ = c.want()
    c.upload()
    c.call()
    dev.sync()
    got = c.got()
    c.free()
    tol = bound(np.where(np.isfinite(want), want, 0), np.nan_to_num(mass), size, q, kv, 64,
                max(lens), new is not None)
    assert np.array_equal(np.isnan(got), np.isnan(want))
    off = np.isinf(want)
    assert np.array_equal(np.isinf(got), off) and np.array_equal(got[off], want[off])
    ok = np.isfinite(want)
    assert (np.abs(got[ok] - want[ok]) <= tol[ok]).all()
    return want


@types
@pytest.mark.parametrize("prompt", [False, True])
@pytest.mark.parametrize("gain", [2.0, 30.0])
def test_infinite_values_that_are_seen(dev, q, kv, prompt, gain):
    """One infinity in a column gives it, two of one sign too, two of both NaN,
    whatever their keys' weights (with a gain of 30 most are below what f32
    holds), in tiles that all rows see and in those that some see."""
    inf, nan = np.inf, np.nan
    put = [(0, 20, 0, 5, inf), (0, 250, 0, 6, -inf), (0, 21, 1, 7, inf), (0, 299, 1, 7, -inf),
           (0, 40, 1, 8, inf), (0, 260, 1, 8, inf), (1, 2, 0, 63, -inf), (1, 30, 1, 0, nan),
           (0, 290, 0, 40, inf)]
    want = seen_not_finite(dev, q, kv, [60, 33] if prompt else None, [300, 40], put_v=put,
                           gain=gain)
    assert np.isinf(want).any() and np.isnan(want).any()


@types
def test_infinite_values_of_a_cache_that_is_cut(dev, q, kv):
    """The parts that workgroups hand to a join."""
    put = [(0, 20, 0, 5, np.inf), (0, 2500, 0, 6, -np.inf), (0, 1500, 1, 7, np.inf),
           (0, 2990, 1, 7, np.inf), (0, 700, 1, 9, np.inf), (0, 2700, 1, 9, -np.inf)]
    for new in (None, [5]):
        for gain in (2.0, 40.0):
            seen_not_finite(dev, q, kv, new, [3000], put_v=put, gain=gain)


@types
def test_infinite_values_of_many_short_sequences(dev, q, kv):
    """Sequences that a wave has to itself, and one after them on the same wave."""
    n = 200
    lens = [20 + i % 90 for i in range(n)]
    c = Case(dev, lens, heads=4, kv_heads=4, dim=64, q=q, kv=kv, seed=3)
    want, mass, size = c.want()
    for s in range(0, n, 7):
        at = 0, c.tables[s, 0], 1, 3, 9
        c.vh[at] = narrow(np.array([-np.inf], np.float32), kv)[0]
        want[s, 1, 9] = -np.inf
    c.upload()
    c.call()
    dev.sync()
    got = c.got()
    c.free()
    tol = bound(np.where(np.isfinite(want), want, 0), mass, size, q, kv, 64, max(lens), False)
    off = np.isinf(want)
    assert off.sum() == 29 and np.array_equal(got[off], want[off])
    assert (np.abs(got[~off] - want[~off]) <= tol[~off]).all()


@types
@pytest.mark.parametrize("prompt", [False, True])
def test_infinite_keys_that_are_seen(dev, q, kv, prompt):
    """A score of -inf has no weight, and the result is finite; one of +inf
    makes it NaN.  Both come of the same key, as the queries' signs are."""
    put = [(0, 20, 0, 9, np.inf), (0, 270, 0, 9, np.inf), (0, 100, 1, 33, -np.inf),
           (1, 20, 0, 3, np.inf)]
    want = seen_not_finite(dev, q, kv, [60, 33] if prompt else None, [300, 40], put_k=put)
    assert np.isnan(want).any() and np.isfinite(want[:1 if not prompt else 60]).any()


@pytest.mark.parametrize("kv", [F16, BF16])
@pytest.mark.parametrize("prompt", [False, True])
def test_infinite_keys_under_small_f32_queries(dev, kv, prompt):
    """The sign of a query's element decides, however small it is beside the
    row's others; the -inf it gives leaves the key out."""
    rows = 60 if prompt else 1
    tiny = [(r, 9, -1e-20 if r % 2 == 0 else -1e-9) for r in range(rows)]
    want = seen_not_finite(dev, F32, kv, [60] if prompt else None, [300], tiny=tiny,
                           put_k=[(0, 20, 0, 9, np.inf), (0, 230, 1, 9, np.inf)])
    assert np.isfinite(want).all()


@types
@pytest.mark.parametrize("prompt", [False, True])
def test_scores_that_are_all_minus_infinity(dev, q, kv, prompt):
    """No key has a weight then: zeros, as for a query that sees none."""
    c = Case(dev, [70, 5], new=[3, 5] if prompt else None, heads=4, kv_heads=2, dim=64, q=q,
             kv=kv)
    c.q[:, :, 9] = -1
    c.qh[:, :, 9] = -1 if q == F32 else narrow(np.array([-1.0]), q)[0]
    for s, n in enumerate([70, 5]):
        for p in range(n):
            c.kh[0, c.tables[s, p // 16], :, p % 16, 9] = narrow(np.array([np.inf]), kv)[0]
    c.upload()
    c.call()
    dev.sync()
    assert not c.got().any()
    c.free()


@types
@pytest.mark.parametrize("prompt", [False, True])
@pytest.mark.parametrize("gap", [14, 18, 21, 23])
@pytest.mark.parametrize("n", [190, 4000])
def test_a_first_key_of_value_zero_that_dominates(dev, q, kv, prompt, n, gap):
    """A first key `gap` nats above all others, its value 0: the result is
    theirs alone.  Over an f16 cache weights, or their last terms, are f16
    numbers, 2^9 or more for the row's largest; their steps below the normal
    range are 2^-24, half of one 2^-25 / 2^9 = 2^-34 of the largest, which is 1
    at most.  That times the value, for each key, comes to the bound."""
    dim = 64
    c = Case(dev, [n], new=[40] if prompt else None, heads=2, kv_heads=1, dim=dim, q=q, kv=kv,
             seed=gap, gain=0.05)
    first = 0, c.tables[0, 0], 0, 0
    rng = np.random.default_rng(gap)
    x = (1000 * (1 + rng.standard_normal(c.v.shape) / 4)).astype(np.float32)
    held = ((c.vh & 0x7fff) != (0x7fc0 if kv == BF16 else 0x7e00))
    bits = narrow(x, kv)
    c.vh[held] = bits[held]
    c.v = (bits.astype(np.uint32) << 16).view(np.float32) if kv == BF16 else \
        bits.view(np.float16).astype(np.float32)
    c.k[..., 0] = 0
    c.kh[..., 0][held[..., 0]] = 0
    c.q[..., 0] = 4
    c.qh[..., 0] = 4 if q == F32 else narrow(np.array([4.0]), q)[0]
    c.v[first], c.vh[first] = 0, 0
    c.k[first] = 0
    c.k[first + (0,)] = gap / 4
    c.kh[first] = narrow(c.k[first], kv)
    want, mass, size = c.want(scale=1.0)
    c.upload()
    c.call(scale=1.0)
    dev.sync()
    got = c.got()
    c.free()
    tol = bound(want, mass, size, q, kv, dim, n, prompt)
    if kv == F16:
        total = sum(np.abs(c.v[0, c.tables[0, p // 16], 0, p % 16]) for p in range(n))
        tol = tol + 2.0 ** -34 * total
    assert want.min() > 0
    assert (np.abs(got - want) <= tol).all(), (np.abs(got / want - 1)).max()


@pytest.mark.parametrize("prompt", [False, True])
def test_scores_at_the_lowest_end_of_f32(dev, prompt):
    """All scores between -3.4e38 and -3e38 in units of log 2: one key's value."""
    for n in (1, 90):
        c = Case(dev, [n], new=[1] if prompt else None, heads=2, kv_heads=1, dim=64, q=F32)
        c.q[:], c.qh[:] = 0, 0
        c.q[..., 3] = c.qh[..., 3] = -2.2e19
        # the first key's score is the largest by 2^120 and more
        k = np.full((n, 64), 1.02e19, np.float32)
        k[0] = 1e19
        for p in range(n):
            c.kh[0, c.tables[0, p // 16], 0, p % 16] = narrow(k[p], BF16)
        c.upload()
        c.call(scale=1.0)
        dev.sync()
        v = c.v[0, c.tables[0, 0], 0, 0]
        assert np.abs(c.got()[0] - v).max() <= 2.0 ** -20 * np.abs(v).max()
        c.free()


@types
@pytest.mark.parametrize("prompt", [False, True])
@pytest.mark.parametrize("sign", [1, -1])
def test_scores_far_past_what_f32_tells_apart(dev, q, kv, prompt, sign):
    """Scores of sizes up to f32's last, all equal (the mean of the values) or
    one above all others by a part of itself (its value): a score's rounding is
    then more than the exponential's whole range."""
    n, dim = 150, 64
    for same in (True, False):
        c = Case(dev, [n], new=[20] if prompt else None, heads=2, kv_heads=1, dim=dim, q=q, kv=kv)
        x = np.zeros(dim, np.float32)
        x[3] = 1.375
        c.qh[:] = x if q == F32 else narrow(x, q)
        for p in range(n):
            k = np.zeros(dim, np.float32)
            k[3] = sign * (0.75 if same or (p == 40) == (sign > 0) else 0.625)
            c.kh[0, c.tables[0, p // 16], 0, p % 16] = narrow(k, kv)
        v = np.stack([c.v[0, c.tables[0, p // 16], 0, p % 16] for p in range(n)])
        rows = range(n - 20, n) if prompt else [n - 1]
        c.upload()
        for e in (10, 18, 19, 20, 21, 22, 23, 24, 25, 26, 27, 28, 29, 30, 31, 40, 80, 125.6):
            for f in (1.0, 1.2345678):
                c.call(scale=f * 2.0 ** e)
                dev.sync()
                got = c.got()
                if same:
                    want = np.stack([v[:p + 1].mean(0, dtype=np.float64) for p in rows])
                    mass = np.stack([np.abs(v[:p + 1]).mean(0, dtype=np.float64) for p in rows])
                else:
                    want = np.broadcast_to(v[40].astype(np.float64), (len(rows), dim))
                    mass = np.abs(want)
                tol = bound(want, mass, np.zeros(len(rows)), q, kv, dim, n, prompt)
                bad = np.abs(got - want[:, None]) > tol[:, None]
                assert np.isfinite(got).all() and not bad.any(), (e, f, same)
        c.free()


@pytest.mark.parametrize("q", [F32, BF16])
@pytest.mark.parametrize("new", [None, [60], [5]])
def test_values_at_the_end_of_bf16(dev, q, new):
    """Sums of weights times values pass f32's range where weights are more than
    1, or keys many; the mean they stand for does not."""
    for n in (300, 3000):
        if new == [60] and n == 3000:
            continue
        for gain in (2.0, 12.0):
            c = Case(dev, [n], new=new, heads=4, kv_heads=2, dim=64, q=q, kv=BF16, seed=n,
                     gain=gain)
            held = c.vh != 0x7fc0
            # magnitudes up to 2^128 (1 - 2^-8), a column of one sign and size
            x = (c.v * np.float32(2.0 ** 125)).clip(-3.38e38, 3.38e38)
            x[..., 7] = 3.38e38
            bits = narrow(x, BF16)
            c.vh[held] = bits[held]
            c.v = (bits.astype(np.uint32) << 16).view(np.float32)
            c.check()


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


@types
@pytest.mark.parametrize("dim", [40, 128, 200])
def test_prompts_of_more_entries_than_a_wave_has_lanes(dev, q, kv, dim):
    """Entries summed up by a launch before: ragged, empty and padded ones,
    chunks after prefixes, a window over some of them."""
    rng = np.random.default_rng(dim)
    n = 150
    new = [int(x) for x in rng.integers(0, 9, n)]
    new[3], new[90] = 70, 41
    lens = [x + int(y) for x, y in zip(new, rng.integers(0, 30, n))]
    lens[90] += 200
    seqs = [int(x) for x in rng.permutation(n)]
    seqs[5] = KV_NONE
    of = {s: new[i] for i, s in enumerate(seqs) if s != KV_NONE}
    for s, x in of.items():
        lens[s] = max(lens[s], x)
    Case(dev, lens, new=new, heads=6, kv_heads=2, dim=dim, page=8, q=q, kv=kv, seqs=seqs,
         extra_rows=3, seed=dim).check(window=60, sinks=5)
    Case(dev, lens, new=new, heads=2, kv_heads=2, dim=dim, page=8, q=q, kv=kv, seqs=seqs,
         seed=dim + 1).check()
