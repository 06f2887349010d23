"""Sample on the GPU against the choice restated in 64 bits (oracle/draft_np.py).

A token may differ only where a border lies nearer to a running sum than the sums'
roundings.  A weight is 2^(i / 16) 2^(r / 16): the exponent's product is off by
2^-53 of up to 2^17, 2^-36 sixteenths of a power of two or 2^-40.5 of the weight,
the series by 2^-42.7 and its rounding by 2^-39, together less than 2^-38.4; a row that
is weighed otherwise has weights rounded by 2^-46 of the largest for each of up to 2^17
logits.  A sum's share is off by no more than its weights', plus that, and the sums of
bins by 2^-52 a step of 10.  The oracle's margin (a share of the whole) is held against
2^-38 and V 2^-46; the inputs here are random, and rows nearer than that are few.  A
logarithm's share is off by a weight's and a sum's part, 2^-37, and rounded to f32
once, half a step of it."""
import math

import numpy as np
import pytest

import accel_amd
from accel_amd import BF16, F16, F32, U32, NO_TOKEN
from oracle import draft_np
from test_gpu_kv_pages import narrow, widen

pytestmark = pytest.mark.gpu
ids = {F32: "f32", F16: "f16", BF16: "bf16"}
types = pytest.mark.parametrize("dtype", [F32, F16, BF16], ids=ids.get)


def draw(dev, x, u, dtype=F32, stream=None, logprobs=True, **opt):
    """Tokens and logarithms of the rows, and the logits as the type holds them."""
    x = np.ascontiguousarray(x, np.float32)
    bits = x if dtype == F32 else narrow(x, dtype)
    rows = x.shape[0]
    held = [dev.upload(bits, dtype), dev.upload(np.asarray(u, np.float32), F32)]
    fill = np.full(rows, 77, np.uint32)
    out, lp = dev.upload(fill, U32), dev.upload(fill.astype(np.float32), F32)
    kw = {}
    for k, v in opt.items():
        v = np.broadcast_to(np.asarray(v, np.uint32 if k == "top_k" else np.float32), (rows,))
        kw[k] = dev.upload(np.ascontiguousarray(v), U32 if k == "top_k" else F32)
    dev.Sample(held[0], held[1], out, lp if logprobs else None, stream=stream, **kw)
    dev.sync(stream)
    res = out.numpy(), lp.numpy()
    for b in held + [out, lp] + list(kw.values()):
        b.free()
    return (*res, x if dtype == F32 else widen(bits, dtype))


def check(dev, x, u, dtype=F32, few=0.03, **opt):
    got, lp, x = draw(dev, x, u, dtype, **opt)
    rows, width = x.shape
    slack = width * 2.0 ** -46 * max(1, width / 2 ** 17) + 2.0 ** -38
    near = 0
    for r in range(rows):
        mine = {k: (np.broadcast_to(v, (rows,))[r]) for k, v in opt.items()}
        # settings as f32 holds them
        mine = {k: int(v) if k == "top_k" else float(np.float32(v)) for k, v in mine.items()}
        token, share, margin = draft_np.sample(x[r], float(np.float32(u[r])), **mine)
        if margin <= slack:
            near += 1
            continue
        assert got[r] == token, (r, got[r], token, margin, mine, u[r])
        assert abs(lp[r] - share) <= 2.0 ** -24 * abs(share) + slack + 2.0 ** -37 or \
            lp[r] == share, (r, lp[r], share)
    assert near <= few * rows


SETTINGS = [dict(), dict(temperature=0.0), dict(temperature=0.7), dict(temperature=1.8),
            dict(top_k=1), dict(top_k=5), dict(top_k=40, temperature=0.8), dict(top_k=3000),
            dict(top_p=0.5), dict(top_p=0.9, temperature=1.3), dict(top_p=0.999),
            dict(min_p=0.05), dict(min_p=0.3, temperature=1.5),
            dict(top_k=50, top_p=0.9), dict(top_k=200, top_p=0.95, min_p=0.02, temperature=0.6),
            dict(top_k=1500, top_p=0.7, temperature=2.0)]


@types
@pytest.mark.parametrize("width", [1, 2, 63, 64, 65, 1000, 1023, 1025, 2049, 4096, 8191, 20011])
def test_widths(dev, dtype, width):
    rng = np.random.default_rng(width)
    rows = 2 * len(SETTINGS)
    x = rng.standard_normal((rows, width)) * 2.5
    x[::3] += 6 * (rng.random((len(x[::3]), width)) < 3 / width)
    kw = {k: [s.get(k, d) for s in SETTINGS] * 2
          for k, d in (("temperature", 1.0), ("top_k", 0), ("top_p", 1.0), ("min_p", 0.0))}
    # 16-bit logits tie, and few weights' sums are the border's where rows are short
    check(dev, x, rng.random(rows), dtype, few=0.1, **kw)


@types
@pytest.mark.parametrize("opt", SETTINGS, ids=str)
def test_settings(dev, dtype, opt):
    rng = np.random.default_rng(len(str(opt)))
    check(dev, rng.standard_normal((12, 32001)) * 3, rng.random(12), dtype, few=0.1, **opt)


@types
@pytest.mark.parametrize("std", [1e-3, 0.05, 0.5, 8.0, 100.0, 1e4])
def test_spreads(dev, dtype, std):
    """Rows nearly flat, whose order has many in little space, and rows that one
    logit has almost wholly."""
    rng = np.random.default_rng(3)
    rows = len(SETTINGS)
    kw = {k: [s.get(k, d) for s in SETTINGS]
          for k, d in (("temperature", 1.0), ("top_k", 0), ("top_p", 1.0), ("min_p", 0.0))}
    check(dev, rng.standard_normal((rows, 12007)) * std, rng.random(rows), dtype, few=0.15, **kw)


@pytest.mark.parametrize("rows", [1, 3, 64, 257, 600])
def test_rows(dev, rows):
    rng = np.random.default_rng(rows)
    pick = rng.integers(0, len(SETTINGS), rows)
    kw = {k: [SETTINGS[i].get(k, d) for i in pick]
          for k, d in (("temperature", 1.0), ("top_k", 0), ("top_p", 1.0), ("min_p", 0.0))}
    check(dev, rng.standard_normal((rows, 5003)) * 3, rng.random(rows), **kw)


@types
def test_a_large_vocabulary(dev, dtype):
    rng = np.random.default_rng(8)
    rows = len(SETTINGS)
    kw = {k: [s.get(k, d) for s in SETTINGS]
          for k, d in (("temperature", 1.0), ("top_k", 0), ("top_p", 1.0), ("min_p", 0.0))}
    check(dev, rng.standard_normal((rows, 262147)) * 3, rng.random(rows), dtype, few=0.15, **kw)


@types
@pytest.mark.parametrize("std", [0.05, 0.5, 2.0])
@pytest.mark.parametrize("rows,width", [(16, 45001), (110, 45001), (16, 230003), (20, 230003),
                                        (16, 300007)])
def test_long_rows_whole_and_in_parts(dev, dtype, std, rows, width):
    """6, 29 and 37 tiles a row, on both sides of where rows are cut, with many logits
    and with few near the borders."""
    rng = np.random.default_rng(rows + width)
    pick = np.arange(rows) % len(SETTINGS)
    kw = {k: [SETTINGS[i].get(k, d) for i in pick]
          for k, d in (("temperature", 1.0), ("top_k", 0), ("top_p", 1.0), ("min_p", 0.0))}
    x = (rng.standard_normal((rows, width), np.float32) * std).astype(np.float32)
    x[1::4, width // 3:width // 3 + 9000] = -np.inf
    check(dev, x, rng.random(rows), dtype, few=0.15, **kw)


def test_a_very_large_row(dev):
    rng = np.random.default_rng(9)
    check(dev, rng.standard_normal((2, (1 << 22) + 3)) * 3, [0.3, 0.6], few=1.0,
          temperature=[0.5, 1.0], top_k=[9, 0])
    got, _, _ = draw(dev, np.zeros((1, 1 << 24), np.float32), [0.75])
    assert got[0] == 3 << 22


@types
def test_equal_logits_go_by_their_index(dev, dtype):
    """Sums of equal weights are whole numbers of them: the borders fall where the
    arithmetic says, and the lower index is first."""
    for c in (0.0, 1.0, -3.5, 12.0):
        for width in (8, 1000, 4096, 50000):
            x = np.full((6, width), c, np.float32)
            got, lp, _ = draw(dev, x, [0, 0.5, 0.75, 0.999, 0.25, 0.5], dtype,
                              top_k=[0, 0, 0, 0, 4, 0], top_p=[1, 1, 1, 0.5, 1, 0.25])
            want = [0, width // 2, width * 3 // 4, math.floor(np.float32(0.999) * (width // 2)),
                    1, width // 8]
            assert got.tolist() == want, (c, width)
            n = [width] * 3 + [width // 2, 4, width // 4]
            assert np.abs(lp + np.log(n)).max() <= 2.0 ** -24 * math.log(width) + 2.0 ** -28


@types
def test_two_values_and_all_rules(dev, dtype):
    # three of 2, the rest of 0 and of -1: e^2, 1 and e^-1 each
    x = np.zeros((1, 40), np.float32)
    x[0, [7, 20, 33]] = 2
    x[0, 30:33] = -1
    for opt, u, want in [(dict(top_k=3), 0.5, 20), (dict(top_k=2), 0.9, 20), (dict(top_k=4), 0.97, 0),
                         (dict(top_k=5), 0.99, 1), (dict(min_p=0.2), 0.99, 33),
                         (dict(min_p=0.1), 0.99, 39), (dict(top_p=0.25), 0.9, 20),
                         (dict(), 0.99999, 32), (dict(temperature=0.0), 0.9, 7)]:
        assert draw(dev, x, [u], dtype, **opt)[0][0] == want, (opt, u)


def test_both_zeros_are_equal(dev):
    x = np.array([[-0.0, 0.0, -0.0, 0.0]], np.float32)
    for u, want in ((0.0, 0), (0.3, 1), (0.6, 2), (0.9, 3)):
        assert draw(dev, x, [u])[0][0] == want
    assert draw(dev, x, [0.9], top_k=2)[0][0] == 1
    assert draw(dev, x, [0.9], temperature=0.0)[0][0] == 0




@types
def test_masked_and_odd_logits(dev, dtype):
    low = {F32: np.finfo(np.float32).min, F16: -65504.0, BF16: -3.3895e38}[dtype]
    rng = np.random.default_rng(5)
    base = rng.standard_normal((1, 3000)).astype(np.float32)
    rows = []
    for fill in (-np.inf, np.nan, low):
        x = base.copy()
        x[0, 1:2000] = fill
        rows.append(x)
    x = np.concatenate(rows)
    # nothing of what is masked is drawn, and the three agree
    for u in (0.0, 0.4, 0.9999):
        for opt in (dict(), dict(top_p=0.9), dict(top_k=1200), dict(min_p=0.01)):
            got, lp, _ = draw(dev, x, [u] * 3, dtype, **opt)
            assert len(set(got.tolist())) == 1 and (got[0] == 0 or got[0] >= 2000)
            assert len(set(lp.tolist())) == 1
    # all masked
    for fill, want in ((-np.inf, NO_TOKEN), (np.nan, NO_TOKEN), (low, 1500)):
        got, lp, _ = draw(dev, np.full((1, 3000), fill, np.float32), [0.5], dtype)
        assert got[0] == want
        assert lp[0] == -np.inf if want == NO_TOKEN else abs(lp[0] + math.log(3000)) < 1e-6
        assert draw(dev, np.full((1, 3000), fill, np.float32), [0.5], dtype, temperature=0.0)[0][0] \
            == (NO_TOKEN if want == NO_TOKEN else 0)
    # one left
    x = np.full((1, 3000), -np.inf, np.float32)
    x[0, 2999] = -50
    for opt in (dict(), dict(top_p=0.1), dict(top_k=7), dict(min_p=1.0), dict(temperature=0.0)):
        got, lp, _ = draw(dev, x, [0.7], dtype, **opt)
        assert got[0] == 2999 and lp[0] == 0
    # infinities share what there is
    x = base.copy()
    x[0, [5, 100, 2000, 2500]] = np.inf
    for u, want in ((0.0, 5), (0.3, 100), (0.6, 2000), (0.99, 2500)):
        for opt in (dict(), dict(min_p=0.5), dict(temperature=0.01)):
            got, lp, _ = draw(dev, x, [u], dtype, **opt)
            assert got[0] == want and abs(lp[0] + math.log(4)) < 1e-6
        assert draw(dev, x, [0.99], dtype, top_k=2)[0][0] == 100
        assert draw(dev, x, [0.99], dtype, top_p=0.5)[0][0] == 100


@types
def test_settings_out_of_range(dev, dtype):
    rng = np.random.default_rng(6)
    x = rng.standard_normal((1, 2000)) * 2
    plain = [draw(dev, x, [u], dtype)[0][0] for u in (0.0, 0.37, 1 - 2.0 ** -24)]
    first = int(draw(dev, x, [0.5], dtype, temperature=0.0)[0][0])
    for t in (-1.0, np.nan, -np.inf, -0.0):
        assert draw(dev, x, [0.9], dtype, temperature=t)[0][0] == first
    for opt in (dict(top_p=1.5), dict(top_p=np.inf), dict(top_p=np.nan), dict(min_p=-1.0),
                dict(min_p=np.nan), dict(top_k=0), dict(top_k=2000), dict(top_k=0xffffffff)):
        assert draw(dev, x, [0.37], dtype, **opt)[0][0] == plain[1], opt
    for opt in (dict(top_p=0.0), dict(top_p=-3.0), dict(top_p=-np.inf), dict(top_k=1),
                dict(top_p=1e-30), dict(temperature=1e-30), dict(temperature=1e-45)):
        assert draw(dev, x, [0.9], dtype, **opt)[0][0] == first, opt
    for u, k in ((-0.5, 0), (np.nan, 0), (-np.inf, 0), (1.0, 2), (7.0, 2), (np.inf, 2)):
        assert draw(dev, x, [u], dtype)[0][0] == plain[k], u
    # all temperatures' end: every logit alike, in their order
    order = np.lexsort((np.arange(2000), -draw(dev, x, [0.5], dtype)[2][0]))
    assert draw(dev, x, [0.25], dtype, temperature=np.inf)[0][0] == order[500]


@pytest.mark.parametrize("scale", [1e-38, 1e-30, 1e30, 3e38])
def test_logits_at_the_ends_of_the_range(dev, scale):
    rng = np.random.default_rng(7)
    x = (rng.uniform(-1, 1, (4, 3001)) * scale).astype(np.float32)
    check(dev, x, [0.2, 0.9, 0.5, 0.7], few=0.3, temperature=[1.0, 3e38, 1.0, 0.5],
          top_p=[1.0, 0.9, 0.5, 1.0])
    check(dev, x, [0.2, 0.9, 0.5, 0.7], few=0.3, temperature=np.float32(scale))


@pytest.mark.parametrize("dtype,step", [(F32, 2.0 ** -149), (BF16, 2.0 ** -133)],
                         ids=["f32", "bf16"])
@pytest.mark.parametrize("steps", [0.5, 2.0, 300.0])
def test_temperatures_of_a_few_of_the_least_steps(dev, dtype, step, steps):
    """Logits that are small multiples of a type's least number, and temperatures to
    match them: what lies between two bins' edges then holds no f32."""
    rng = np.random.default_rng(11)
    rows = 8
    x = np.round(rng.standard_normal((rows, 20000)) * 3 * steps) * step
    t = max(step * steps, 2.0 ** -149)
    check(dev, x.astype(np.float32), rng.random(rows), dtype, few=0.3, temperature=t,
          top_p=[1, 0.9, 0.5, 1, 0.8, 1, 1, 0.95], top_k=[0, 0, 0, 700, 50, 1, 0, 0],
          min_p=[0, 0, 0, 0, 0, 0, 0.1, 0.01])


def test_far_from_zero(dev):
    """Weights go by the distance to the largest, however far from zero both are."""
    rng = np.random.default_rng(17)
    x = (np.round(rng.standard_normal((8, 9000)) * 64) / 16 + 4096).astype(np.float32)
    u = rng.random(8)
    for opt in (dict(), dict(temperature=0.01), dict(top_p=0.8), dict(top_k=30, min_p=0.01)):
        a, b = draw(dev, x, u, **opt), draw(dev, x - 4096, u, **opt)
        assert np.array_equal(a[0], b[0]), opt
        assert np.abs(a[1] - b[1]).max() <= 2.0 ** -23 * np.abs(b[1]).max()
        check(dev, x, u, few=0.5, **opt)


def test_chances(dev):
    """Random numbers spread evenly give each token as often as its share says: a
    row's tokens ascend through the order with u, and each has the share of the
    numbers that its logarithm says, to one of them at either end."""
    rng = np.random.default_rng(12)
    n, width = 4096, 50
    row = rng.standard_normal(width) * 2
    u = (np.arange(n) + 0.5) / n
    got, lp, x = draw(dev, np.tile(row, (n, 1)), u, top_p=0.97)
    order = np.lexsort((np.arange(width), -x[0]))
    rank = np.argsort(order)[got]
    assert (np.diff(rank) >= 0).all()
    for t in np.unique(got):
        often = (got == t).sum()
        assert abs(often - n * math.exp(lp[got == t][0])) <= 1 + n * 1e-6
    assert abs(sum(math.exp(lp[got == t][0]) for t in np.unique(got)) - 1) <= \
        (width - len(np.unique(got))) / n + 1e-6


def test_a_row_of_no_matrix_and_no_rows(dev):
    x = dev.upload(np.array([0.0, 3.0, 1.0], np.float32))
    u, out = dev.upload(np.array([0.1], np.float32)), dev.upload(np.array([9], np.uint32))
    dev.Sample(x, u, out)
    dev.sync()
    assert out.numpy()[0] == 1
    none = [accel_amd.Buffer(dev, 0, 0, t, s)
            for t, s in ((F32, (0, 3)), (F32, (0,)), (U32, (0,)))]
    dev.Sample(*none)
    dev.sync()


def test_odd_addresses(dev):
    """Rows of an odd width start at every alignment of their type."""
    rng = np.random.default_rng(13)
    for dtype, size in ((F32, 4), (F16, 2), (BF16, 2)):
        x = rng.standard_normal(4 * 1237 + 8).astype(np.float32) * 2
        bits = x if dtype == F32 else narrow(x, dtype)
        whole = dev.upload(bits, dtype)
        u = np.array([0.1, 0.5, 0.7, 0.95], np.float32)
        for at in range(8):
            part = accel_amd.Buffer(dev, whole.ptr + at * size, 4 * 1237 * size, dtype, (4, 1237))
            ub, out = dev.upload(u), dev.upload(np.zeros(4, np.uint32))
            dev.Sample(part, ub, out)
            dev.sync()
            want = draw(dev, x[at:at + 4 * 1237].reshape(4, 1237), u, dtype)[0]
            assert np.array_equal(out.numpy(), want)
            for b in (ub, out):
                b.free()
        whole.free()


@types
def test_replays_and_streams(dev, dtype):
    """Captured once on a stream of its own and replayed over other logits, beside
    another captured call on the same workspace, eager calls between."""
    rng = np.random.default_rng(14)
    st = dev.stream()
    sets = []
    for rows, width in ((3, 40009), (70, 3001)):
        x = rng.standard_normal((rows, width)) * 3
        bits = lambda v: v.astype(np.float32) if dtype == F32 else narrow(  # noqa: E731
            v.astype(np.float32), dtype)
        b = dict(x=dev.upload(bits(x), dtype), u=dev.upload(rng.random(rows).astype(np.float32)),
                 out=dev.upload(np.zeros(rows, np.uint32)), k=dev.upload(np.full(rows, 90, np.uint32)),
                 p=dev.upload(np.full(rows, 0.9, np.float32)))
        call = lambda b=b: dev.Sample(b["x"], b["u"], b["out"], top_k=b["k"], top_p=b["p"],  # noqa: E731
                                      stream=st)
        call()
        dev.sync(st)
        dev.capture_begin(st)
        call()
        sets.append((b, bits, rows, width, dev.capture_end(st)))
    for _ in range(3):
        for b, bits, rows, width, ex in sets:
            x = (rng.standard_normal((rows, width)) * 3).astype(np.float32)
            b["x"].write(bits(x))
            b["out"].write(np.full(rows, 5, np.uint32))
            dev.launch(ex, st)
            dev.sync(st)
            want = draw(dev, x, b["u"].numpy(), dtype, top_k=90, top_p=0.9)[0]
            assert np.array_equal(b["out"].numpy(), want)
    for b, _, _, _, ex in sets:
        dev.destroy_exec(ex)
        for v in b.values():
            v.free()
    dev.destroy_stream(st)


def test_calls_repeat_themselves(dev):
    rng = np.random.default_rng(15)
    x = rng.standard_normal((40, 30011)) * 1.5
    u = rng.random(40)
    first = draw(dev, x, u, top_p=0.9, logprobs=True)
    for _ in range(4):
        again = draw(dev, x, u, top_p=0.9)
        assert np.array_equal(first[0], again[0]) and np.array_equal(first[1], again[1])
    # rows in parts, whichever of them ends last
    x = rng.standard_normal((5, 150001)) * 1.5
    first = draw(dev, x, u[:5], top_p=0.9)
    for _ in range(4):
        again = draw(dev, x, u[:5], top_p=0.9)
        assert np.array_equal(first[0], again[0]) and np.array_equal(first[1], again[1])
    x = rng.standard_normal((40, 30011)) * 1.5
    first = draw(dev, x, u, top_p=0.9)
    # the logarithms are asked for or not
    assert np.array_equal(draw(dev, x, u, top_p=0.9, logprobs=False)[0], first[0])
