"""The checks of arguments of drafts' attention, sampling, acceptance and keeping
(CPU: every check runs before a device is touched)."""
import ctypes

import pytest

import accel_amd
from accel_amd import BF16, F16, F32, I8, U32, SamplingDesc
from test_kv_refusals import A, L, R, cache, refused, tensor


def tree(q=None, off=None, par=None, c=None, layer=0, seqs=None, opt=None, out=None):
    q = q or tensor((6, 4, 64), BF16)
    return L.accel_paged_tree_attention(
        0, None, R(q), R(off or tensor((3,))), R(par or tensor((6,))) if par != 0 else None,
        R(c or cache()), layer, seqs, opt, R(out or q))


def test_tree_attention():
    refused(tree(par=0), "PagedTreeAttention", "parents")
    refused(tree(par=tensor((5,))), "parents", "5 entries")
    refused(tree(par=tensor((6,), F32)), "parents")
    refused(tree(par=tensor((6,), data=0)), "parents is missing")
    refused(tree(off=tensor((0,))), "offsets")
    refused(tree(q=tensor((6, 3, 64), BF16)), "[6 3 64]")
    refused(tree(q=tensor((6, 4, 64), F16)), "f16")
    refused(tree(layer=3), "layer 3")
    refused(tree(out=tensor((6, 4, 64), F32)), "output")
    refused(tree(c=cache(page_size=12)), "pages of 12")
    refused(tree(off=tensor((9,))), "8 entries")
    refused(tree(opt=R(accel_amd.AttentionDesc(-1.0, 0, 0))), "scale")
    refused(tree(opt=R(accel_amd.AttentionDesc(1.0, -1, 0))), "window")
    refused(L.accel_paged_tree_attention(0, None, None, R(tensor((3,))), R(tensor((6,))),
                                         R(cache()), 0, None, None, None), "queries are missing")


def sample(x=None, u=0, tokens=0, logprobs=None, **opt):
    x = x or tensor((5, 100), F32)
    u = tensor((5,), F32) if u == 0 else u
    tokens = tensor((5,)) if tokens == 0 else tokens
    d = SamplingDesc(*(ctypes.pointer(opt[k]) if k in opt else None
                       for k in ("temperature", "top_k", "top_p", "min_p")))
    ref = lambda t: None if t is None else R(t)  # noqa: E731
    return L.accel_sample(0, None, R(x), ref(u), R(d), ref(tokens), ref(logprobs))


def test_sample():
    refused(sample(x=tensor((5, 100), I8)), "Sample", "i8")
    refused(sample(x=tensor((5, 1, 100), F32)), "[rows, width]")
    refused(sample(x=tensor((5, 0), F32)), "[5 0]")
    refused(sample(x=tensor((5, (1 << 24) + 1), F32)), "rows of 1 to 16777216")
    refused(sample(x=tensor((1 << 31, 100), F32)), "rows")
    refused(sample(x=tensor((5, 100), F32, 0)), "logits are missing")
    refused(sample(u=None), "random numbers")
    refused(sample(u=tensor((4,), F32)), "random numbers", "5")
    refused(sample(u=tensor((5,), F16)), "random numbers")
    refused(sample(u=tensor((5,), F32, 0)), "random numbers is missing")
    refused(sample(tokens=None), "tokens")
    refused(sample(tokens=tensor((5,), F32)), "tokens")
    refused(sample(tokens=tensor((6,))), "tokens")
    refused(sample(logprobs=tensor((5,), U32)), "logarithms")
    for k, t in (("temperature", F32), ("top_k", U32), ("top_p", F32), ("min_p", F32)):
        refused(sample(**{k: tensor((4,), t)}), k)
        refused(sample(**{k: tensor((5,), F32 if t == U32 else U32)}), k)
        refused(sample(**{k: tensor((5, 1), t)}), k)
        refused(sample(**{k: tensor((5,), t, 0)}), k, "missing")
    refused(L.accel_sample(0, None, None, None, None, None, None), "logits")


def accept(**kw):
    d = dict(tokens=tensor((6,)), parents=tensor((6,)), offsets=tensor((3,)),
             sampled=tensor((6,)), path=tensor((2, 4)), counts=tensor((2,)), next=tensor((2,)))
    d.update(kw)
    return L.accel_tree_accept(0, None, *(None if t is None else R(t) for t in d.values()))


@pytest.mark.parametrize("name", ["tokens", "parents", "offsets", "sampled", "path", "counts",
                                  "next"])
def test_accept_without_a_list(name):
    refused(accept(**{name: None}), "TreeAccept")


def test_accept():
    refused(accept(parents=tensor((5,))), "parents")
    refused(accept(sampled=tensor((7,))), "sampled")
    refused(accept(tokens=tensor((6,), F32)), "tokens")
    refused(accept(offsets=tensor((0,))), "offsets")
    refused(accept(path=tensor((3, 4))), "paths")
    refused(accept(path=tensor((2, 0))), "paths")
    refused(accept(path=tensor((2, 4097))), "paths")
    refused(accept(path=tensor((8,))), "paths")
    refused(accept(path=tensor((2, 4), data=0)), "paths are missing")
    refused(accept(counts=tensor((1,))), "counts")
    refused(accept(next=tensor((3,))), "next")
    n = 1 << 20
    refused(accept(offsets=tensor((n + 1,)), path=tensor((n, 4096)), counts=tensor((n,)),
                   next=tensor((n,))), "31-bit")


def keep(c=None, seqs=None, offsets=None, path=None, counts=None):
    return L.accel_kv_keep(0, None, R(c or cache()), seqs, R(offsets or tensor((3,))),
                           R(path or tensor((2, 4))), R(counts or tensor((2,))))


def test_keep():
    refused(keep(c=cache(dtype=F32)), "KVKeep", "f32")
    refused(L.accel_kv_keep(0, None, None, None, None, None, None), "KVKeep", "needs keys")
    refused(L.accel_kv_keep(0, None, R(cache()), None, None, None, None), "offsets")
    refused(keep(path=tensor((2, 4), F32)), "paths")
    refused(keep(path=tensor((1, 4))), "paths")
    refused(keep(counts=tensor((3,))), "counts")
    refused(keep(seqs=R(tensor((3,)))), "sequences")
    refused(keep(offsets=tensor((6,)), path=tensor((5, 4)), counts=tensor((5,))), "5 entries")
