"""The paged cache's and its attention's checks of arguments (CPU: every check
runs before a device is touched)."""
import ctypes

import pytest

import accel_amd
from accel_amd import BF16, F16, F32, I8, U32, AttentionDesc, KVCacheDesc, Tensor

A = 1 << 20          # an aligned address that no call here reaches


def cache(**kw):
    d = dict(keys=A, values=A, refs=A, tables=A, lens=A, dtype=BF16, kv_heads=2, page_size=16,
             head_dim=64, layers=3, pages=10, sequences=4, slots=5)
    d.update(kw)
    return KVCacheDesc(**d)


def tensor(shape, dtype=U32, data=A):
    t = Tensor(data, dtype, len(shape))
    for i, n in enumerate(shape):
        t.shape[i] = n
    return t


def refused(rc, *words):
    assert rc == accel_amd.E_INVALID, (rc, accel_amd.last_error())
    msg = accel_amd.last_error()
    assert msg.startswith("accel/tensor: "), msg
    for w in words:
        assert w in msg, (w, msg)


L = accel_amd.lib()
R = ctypes.byref


@pytest.mark.parametrize("bad,word", [
    (dict(keys=0), "needs keys"), (dict(values=None), "needs keys"), (dict(refs=0), "refs"),
    (dict(tables=0), "tables"), (dict(lens=0), "lens"),
    (dict(dtype=F32), "f32"), (dict(dtype=I8), "i8"), (dict(dtype=99), "unknown"),
    (dict(page_size=0), "pages of 0"), (dict(page_size=24), "pages of 24"),
    (dict(page_size=4), "pages of 4"), (dict(page_size=8192), "pages of 8192"),
    (dict(head_dim=0), "heads of 0"), (dict(head_dim=68), "heads of 68"),
    (dict(head_dim=264), "heads of 264"), (dict(kv_heads=0), "0 key-value"),
    (dict(layers=0), "0 layers"), (dict(pages=0), "0 pages"), (dict(pages=1 << 31), "pages"),
    (dict(sequences=0), "0 sequences"), (dict(slots=-1), "slots"),
    (dict(slots=1 << 28), "31 bits"), (dict(sequences=1 << 20, slots=1 << 12), "31 bits"),
    (dict(pages=2 ** 31 - 1, layers=60000, kv_heads=4096, page_size=4096, head_dim=256,
          slots=1), "address space"),
    (dict(keys=A + 2), "aligned"), (dict(values=A + 8), "aligned"),
])
def test_every_entry_refuses_a_cache_it_cannot_serve(bad, word):
    c = cache(**bad)
    q = tensor((4, 2, 64), BF16)
    u = tensor((4,))
    calls = [
        lambda: L.accel_kv_clear(0, None, R(c)),
        lambda: L.accel_kv_reserve(0, None, R(c), None, R(u)),
        lambda: L.accel_kv_append(0, None, R(c), 0, R(q), R(q), None, None),
        lambda: L.accel_kv_fork(0, None, R(c), R(u), R(u)),
        lambda: L.accel_kv_trim(0, None, R(c), None, 5, 0),
        lambda: L.accel_kv_free(0, None, R(c), None),
        lambda: L.accel_kv_compact(0, None, R(c), None),
        lambda: L.accel_kv_copy(0, None, R(c), R(u), R(u)),
        lambda: L.accel_paged_attention(0, None, R(q), R(c), 0, None, None, R(q)),
        lambda: L.accel_paged_prefill(0, None, R(q), R(u), R(c), 0, None, None, R(q)),
    ]
    for call in calls:
        refused(call(), word)


def test_a_missing_cache():
    refused(L.accel_kv_clear(0, None, None), "KVClear", "needs keys")
    refused(L.accel_kv_compact(0, None, None, None), "KVCompact")


@pytest.mark.parametrize("grow,seqs,word", [
    (None, None, "grow"), (tensor((4,), F32), None, "grow"), (tensor((2, 2)), None, "grow"),
    (tensor((3,)), None, "grow has 3"), (tensor((4,), U32, 0), None, "grow is missing"),
    (tensor((3,)), tensor((2,)), "sequences has 2"), (tensor((3,)), tensor((3,), I8), "sequences"),
    (tensor((-1,)), tensor((-1,)), "grow"),
])
def test_reserve(grow, seqs, word):
    refused(L.accel_kv_reserve(0, None, R(cache()), R(seqs) if seqs else None,
                               R(grow) if grow else None), "KVReserve", word)


@pytest.mark.parametrize("layer,k,v,seqs,offsets,word", [
    (-1, (4, 2, 64), (4, 2, 64), None, None, "layer -1"),
    (3, (4, 2, 64), (4, 2, 64), None, None, "layer 3 of a cache of 3"),
    (0, (4, 3, 64), (4, 3, 64), None, None, "2 heads of 64"),
    (0, (4, 2, 32), (4, 2, 32), None, None, "2 heads of 64"),
    (0, (4, 2, 64), (3, 2, 64), None, None, "values [3 2 64]"),
    (0, (4, 128), (4, 128), None, None, "keys [4 128]"),
    (0, (5, 2, 64), (5, 2, 64), None, None, "5 entries"),
    (0, (4, 2, 64), (4, 2, 64), (3,), None, "sequences has 3"),
    (0, (4, 2, 64), (4, 2, 64), None, (0,), "offsets"),
    (0, (4, 2, 64), (4, 2, 64), None, (6,), "5 entries"),
    (0, (4, 2, 64), (4, 2, 64), (2,), (4,), "sequences has 2"),
])
def test_append(layer, k, v, seqs, offsets, word):
    t = [R(tensor(x)) if x else None for x in (seqs, offsets)]
    refused(L.accel_kv_append(0, None, R(cache()), layer, R(tensor(k, F32)), R(tensor(v, F32)), *t),
            "KVAppend", word)


def test_append_types_and_addresses():
    c, ok = cache(), tensor((4, 2, 64), F32)
    call = lambda k, v: L.accel_kv_append(0, None, R(c), 0, R(k), R(v), None, None)  # noqa: E731
    refused(call(tensor((4, 2, 64), F16), ok), "keys are f16 and values f32")
    refused(call(tensor((4, 2, 64), I8), tensor((4, 2, 64), I8)), "i8")
    refused(call(ok, tensor((4, 2, 64), F32, 0)), "missing")
    refused(call(ok, tensor((4, 2, 64), F32, A + 4)), "aligned")
    refused(L.accel_kv_append(0, None, R(c), 0, R(ok), None, None, None), "missing")


def test_fork_copy_and_free():
    c, u = cache(), tensor((4,))
    refused(L.accel_kv_fork(0, None, R(c), R(u), R(tensor((3,)))), "children has 3")
    refused(L.accel_kv_fork(0, None, R(c), None, R(u)), "parents")
    refused(L.accel_kv_fork(0, None, R(c), R(u), None), "children")
    refused(L.accel_kv_copy(0, None, R(c), R(u), R(tensor((5,)))), "target pages has 5")
    refused(L.accel_kv_copy(0, None, R(c), R(tensor((4,), F32)), R(u)), "source pages")
    big = tensor((1 << 30,))
    refused(L.accel_kv_copy(0, None, R(c), R(big), R(big)), "31-bit grid")
    refused(L.accel_kv_fork(0, None, R(c), R(big), R(big)), "31-bit grid")
    refused(L.accel_kv_free(0, None, R(c), R(tensor((2, 2)))), "u32 vector")
    refused(L.accel_kv_trim(0, None, R(c), None, 0, 0), "window of 0")
    refused(L.accel_kv_trim(0, None, R(c), None, 4, -1), "-1 sinks")
    refused(L.accel_kv_compact(0, None, R(c), R(tensor((2,)))), "live has 2")


@pytest.mark.parametrize("q,out,word", [
    ((4, 3, 64), (4, 3, 64), "multiple"), ((4, 0, 64), (4, 0, 64), "multiple"),
    ((4, 4, 32), (4, 4, 32), "heads of 64"), ((4, 256), (4, 256), "[4 256]"),
    ((4, 4, 64), (3, 4, 64), "output"), ((5, 4, 64), (5, 4, 64), "5 entries"),
    ((1 << 30, 4, 64), (1 << 30, 4, 64), "31-bit grid"),
])
def test_attention_shapes(q, out, word):
    c = cache()
    refused(L.accel_paged_attention(0, None, R(tensor(q, F32)), R(c), 0, None, None,
                                    R(tensor(out, F32))), "PagedAttention", word)


def test_attention_types_options_and_lists():
    c, q = cache(), tensor((4, 4, 64), BF16)

    def call(q=q, out=None, layer=0, seqs=None, **opt):
        o = AttentionDesc(**opt)
        return L.accel_paged_attention(0, None, R(q), R(c), layer, seqs, R(o), R(out or q))

    refused(call(tensor((4, 4, 64), F16)), "f16", "bf16")
    refused(call(out=tensor((4, 4, 64), F32)), "output")
    refused(call(layer=3), "layer 3")
    refused(call(scale=-1.0), "scale -1")
    refused(call(scale=float("nan")), "finite")
    refused(call(scale=float("inf")), "finite")
    refused(call(window=-1), "window -1")
    refused(call(sinks=-1), "sinks -1")
    refused(call(tensor((4, 4, 64), BF16, A + 8)), "aligned")
    refused(call(tensor((4, 4, 64), BF16, 0)), "missing")
    refused(call(seqs=R(tensor((3,)))), "sequences has 3")
    f = lambda off, seqs=None: L.accel_paged_prefill(  # noqa: E731
        0, None, R(q), off, R(c), 0, seqs, None, R(q))
    refused(f(None), "PagedPrefill", "offsets")
    refused(f(R(tensor((0,)))), "offsets")
    refused(f(R(tensor((7,)))), "6 entries")
    refused(f(R(tensor((3,))), R(tensor((3,)))), "sequences has 3")
    refused(L.accel_paged_prefill(0, None, None, R(tensor((3,))), R(c), 0, None, None, R(q)),
            "queries are missing")


def test_a_freed_cache_is_refused():
    class Held:
        ptr, dtype, shape = A, BF16, (1, 4, 2, 16, 64)

        def free(self):
            self.ptr = 0

    k = Held()
    b = lambda shape: accel_amd.Buffer(None, 0, 0, U32, shape)  # noqa: E731
    c = accel_amd.KVCache(None, k, k, b((4,)), b((3, 2)), b((3,)))
    c.free()
    refused(L.accel_kv_clear(0, None, R(c.desc())), "needs keys")


def test_a_closed_device_is_named():
    rc = L.accel_kv_clear(63, None, R(cache()))
    assert rc == accel_amd.E_NO_DEVICE, accel_amd.last_error()
    q = tensor((4, 4, 64), BF16)
    rc = L.accel_paged_attention(63, None, R(q), R(cache()), 0, None, None, R(q))
    assert rc == accel_amd.E_NO_DEVICE


def test_the_binding_checks_a_caches_shapes():
    b = lambda shape, t=U32: accel_amd.Buffer(None, A, 0, t, shape)  # noqa: E731
    k = b((1, 4, 2, 16, 64), BF16)
    good = dict(keys=k, values=k, refs=b((4,)), tables=b((3, 2)), lens=b((3,)))
    d = accel_amd.KVCache(None, **good).desc()
    assert (d.layers, d.pages, d.kv_heads, d.page_size, d.head_dim, d.sequences, d.slots) == \
        (1, 4, 2, 16, 64, 3, 2)
    for key, bad in [("keys", b((4, 2, 16, 64), BF16)), ("values", b((1, 4, 2, 16, 64), F16)),
                     ("refs", b((5,))), ("tables", b((3,))), ("lens", b((2,))),
                     ("lens", b((3,), F32))]:
        with pytest.raises(ValueError):
            accel_amd.KVCache(None, **{**good, key: bad})
