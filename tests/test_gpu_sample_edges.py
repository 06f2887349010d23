"""Sample where a call takes another way than the usual: rows of parts in several launches,
more rows than a launch has, rows whose first logits are masked, rows of millions, against
the choice in 64 bits (oracle/draft_np.py) within the bounds of test_gpu_sample.py."""
import math

import numpy as np
import pytest

import accel_amd
from accel_amd import BF16, F16, F32
from oracle import draft_np
from test_gpu_kv_pages import narrow
from test_gpu_sample import SETTINGS, check, draw, types

pytestmark = pytest.mark.gpu


def settings(rows):
    pick = [SETTINGS[i % len(SETTINGS)] for i in range(rows)]
    return {k: np.array([s.get(k, d) for s in pick])
            for k, d in (("temperature", 1.0), ("top_k", 0), ("top_p", 1.0), ("min_p", 0.0))}


def test_rows_in_parts_in_several_launches(dev):
    """262 rows of 33 parts each take two launches of up to 248 rows over one workspace:
    they give what calls of one launch give, bit for bit, again and again, and the rows on
    both sides of the cut what the definition gives."""
    rng = np.random.default_rng(20)
    rows, width = 262, 262144
    x = rng.standard_normal((rows, width), np.float32) * 2
    x[3::7, 100:200000] = -np.inf
    u, kw = rng.random(rows), settings(rows)
    want = [draw(dev, x[a:b], u[a:b], BF16, **{k: v[a:b] for k, v in kw.items()})
            for a, b in ((0, 131), (131, rows))]
    for _ in range(3):
        got = draw(dev, x, u, BF16, **kw)
        for i in range(2):
            assert np.array_equal(got[i], np.concatenate([w[i] for w in want]))
    near = np.r_[0:4, 240:rows]
    check(dev, x[near], u[near], BF16, few=0.15, **{k: v[near] for k, v in kw.items()})


def test_more_rows_than_a_launch_has(dev):
    """A few more than 2^22 rows of three logits."""
    rng = np.random.default_rng(21)
    rows = (1 << 22) + 5
    x = rng.standard_normal((rows, 3)).astype(np.float32)
    u = rng.random(rows).astype(np.float32)
    got, lp, _ = draw(dev, x, u)
    order = np.argsort(-x, 1, kind="stable")
    w = np.exp(np.take_along_axis(x, order, 1).astype(np.float64) - x.max(1, keepdims=True))
    run = np.cumsum(w, 1) / w.sum(1, keepdims=True)
    j = (run <= u[:, None]).sum(1)
    clear = np.abs(run - u[:, None]).min(1) > 2.0 ** -37
    assert clear.mean() > 0.999
    token = np.take_along_axis(order, np.minimum(j, 2)[:, None], 1)[:, 0]
    assert np.array_equal(got[clear], token[clear])
    share = np.log(np.take_along_axis(w, np.minimum(j, 2)[:, None], 1)[:, 0] / w.sum(1))
    assert (np.abs(lp - share) <= 2.0 ** -24 * np.abs(share) + 2.0 ** -36)[clear].all()


@types
@pytest.mark.parametrize("fill", ["-inf", "nan", "lowest", -60000.0, -300.0])
@pytest.mark.parametrize("rows,width,masked", [
    (16, 9001, 4096), (16, 20011, 5000), (16, 32001, 31990), (64, 100003, 4097),
    (64, 100003, 99990), (16, 100003, 60000)])
def test_rows_whose_start_is_masked(dev, dtype, fill, rows, width, masked):
    """The first logits, more than a workgroup reads at first, have no place beside the
    rest: none at all, or one that is far below."""
    rng = np.random.default_rng(masked)
    low = {F32: np.finfo(np.float32).min, F16: -65504.0, BF16: -3.3895e38}[dtype]
    value = {"-inf": -np.inf, "nan": np.nan, "lowest": low}.get(fill, fill)
    x = (rng.standard_normal((rows, width), np.float32) * 3).astype(np.float32)
    x[:, :masked] = value
    u, kw = rng.random(rows), settings(rows)
    # rows of more are told apart by the same rules; 16 of each are compared
    some = np.arange(rows) if rows <= 16 else np.r_[0:8, rows - 8:rows]
    got = draw(dev, x, u, dtype, **kw)
    again = draw(dev, x[some], u[some], dtype, **{k: v[some] for k, v in kw.items()})
    for i in range(2):
        assert np.array_equal(got[i][some], again[i])
    assert (got[0] >= masked).all()
    check(dev, x[some], u[some], dtype, few=0.15, **{k: v[some] for k, v in kw.items()})


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("opt", [dict(), dict(temperature=0.7), dict(top_p=0.9),
                                 dict(temperature=1.5, min_p=1e-4), dict(top_k=100000)], ids=str)
def test_rows_of_millions(dev, dtype, opt):
    """Every token is held to the definition: a weight is off by 2^-38.4 of itself, what
    lies 46 factors of two below the largest is left out, and the oracle's own sums of n
    terms are off by n 2^-53."""
    rng = np.random.default_rng(22)
    rows, width = 3, (1 << 22) + 3
    x = (rng.standard_normal((rows, width), np.float32) * 3).astype(np.float32)
    u = rng.random(rows)
    got, lp, x = draw(dev, x, u, dtype, **opt)
    for r in range(rows):
        mine = {k: v if k == "top_k" else float(np.float32(v)) for k, v in opt.items()}
        e = (x[r].astype(np.float64) - x[r].max()) / mine.get("temperature", 1.0)
        w, kept = np.exp(e), x[r]
        least = mine.pop("min_p", 0.0)
        if least:
            # a weight is held against this one alone, of which its error is 2^-38.4
            assert np.abs(w - least).min() > 2.0 ** -38 * least
            kept = np.where(w >= least, kept, -np.inf)
        token, share, margin = draft_np.sample(kept, float(np.float32(u[r])), **mine)
        left_out = w[e < -45.9 * math.log(2)].sum() / w.sum()
        slack = 2.0 ** -37 + left_out + width * 2.0 ** -53
        assert margin > slack
        assert got[r] == token
        assert abs(lp[r] - share) <= 2.0 ** -24 * abs(share) + 4 * slack


@pytest.mark.parametrize("rows,width", [(260, 1 << 24), (140000, 32001)])
def test_logits_past_32_bits(dev, rows, width):
    """More than 2^32 logits, in parts and whole: the first and the last rows give what
    they give alone, bit for bit (the others are whatever memory held, at a temperature of
    0)."""
    rng = np.random.default_rng(23)
    some = [0, rows - 2, rows - 1]
    x = (rng.standard_normal((3, width), np.float32) * 3).astype(np.float32)
    u = rng.random(3).astype(np.float32)
    kw = dict(temperature=[0.8, 0.8, 0.9], top_k=[40, 0, 0], top_p=[0.9, 1.0, 0.8])
    want = draw(dev, x, u, BF16, **kw)
    logits = dev.alloc((rows, width), BF16)
    bits = narrow(x, BF16)
    for i, r in enumerate(some):
        accel_amd._check(accel_amd.lib().accel_hip_write(
            dev.index, logits.ptr, r * width * 2, bits[i].ctypes.data, bits[i].nbytes))
    full = {k: np.zeros(rows, np.float32) for k in ("u", "temperature", "top_p", "lp")}
    full["top_k"], full["token"] = np.zeros(rows, np.uint32), np.zeros(rows, np.uint32)
    full["u"][some] = u
    for k, v in kw.items():
        full[k][some] = v
    b = {k: dev.upload(v) for k, v in full.items()}
    dev.Sample(logits, b["u"], b["token"], b["lp"], temperature=b["temperature"],
               top_k=b["top_k"], top_p=b["top_p"])
    dev.sync()
    assert np.array_equal(b["token"].numpy()[some], want[0])
    assert np.array_equal(b["lp"].numpy()[some], want[1])
    for x in [logits, *b.values()]:
        x.free()
