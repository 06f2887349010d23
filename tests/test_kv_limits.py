"""Sizes at the ends of what the paged cache's calls count in (CPU: every check
runs before a device is touched)."""
import pytest

import accel_amd
from accel_amd import BF16, AccelError, AttentionDesc
from test_kv_refusals import A, L, R, cache, refused, tensor

MOST = 2 ** 31 - 1 - 1024


@pytest.mark.parametrize("n", [MOST + 1, 2 ** 31 - 2, 2 ** 31 - 1, 2 ** 40])
def test_lists_longer_than_the_kernels_step_over(n):
    c, u = cache(), tensor((n,))
    q = tensor((4, 2, 64), BF16)
    refused(L.accel_kv_reserve(0, None, R(c), R(u), R(u)), f"grow has {n}", f"up to {MOST}")
    refused(L.accel_kv_free(0, None, R(c), R(u)), f"sequences has {n}")
    refused(L.accel_kv_trim(0, None, R(c), R(u), 5, 0), f"sequences has {n}")
    refused(L.accel_kv_fork(0, None, R(c), R(u), R(u)), f"parents has {n}")
    refused(L.accel_kv_copy(0, None, R(c), R(u), R(u)), f"pages has {n}")
    refused(L.accel_kv_append(0, None, R(c), 0, R(q), R(q), None, R(u)), f"offsets has {n}")
    refused(L.accel_paged_prefill(0, None, R(q), R(u), R(c), 0, None, None, R(q)),
            f"offsets has {n}")


def test_the_longest_lists_pass_the_checks():
    # a device that is not open is the first thing found wrong
    c, u = cache(), tensor((MOST,))
    q = tensor((4, 2, 64), BF16)
    s = tensor((MOST - 1,))
    for rc in (L.accel_kv_reserve(63, None, R(c), R(u), R(u)),
               L.accel_kv_free(63, None, R(c), R(u)),
               L.accel_kv_append(63, None, R(c), 0, R(q), R(q), R(s), R(u)),
               L.accel_paged_prefill(63, None, R(q), R(u), R(c), 0, R(s), None, R(q))):
        assert rc == accel_amd.E_NO_DEVICE, accel_amd.last_error()


def test_scales_that_pass_the_range_in_units_of_log_2():
    c, q, off = cache(), tensor((4, 4, 64), BF16), tensor((5,))
    for scale in (3.4e38, 2.4e38, 1.8e38):
        o = AttentionDesc(scale, 0, 0)
        refused(L.accel_paged_attention(63, None, R(q), R(c), 0, None, R(o), R(q)), "2^127")
        refused(L.accel_paged_prefill(63, None, R(q), R(off), R(c), 0, None, R(o), R(q)), "2^127")
    o = AttentionDesc(2.0 ** 127, 0, 0)
    rc = L.accel_paged_attention(63, None, R(q), R(c), 0, None, R(o), R(q))
    assert rc == accel_amd.E_NO_DEVICE


def test_a_cache_that_is_refused_keeps_no_memory():
    class Held:
        def __init__(self, shape, dtype):
            self.shape, self.dtype, self.ptr = shape, dtype, A
            held.append(self)

        def free(self):
            self.ptr = 0

    held = []
    dev = accel_amd.Device.__new__(accel_amd.Device)
    dev.index, dev.alloc = 63, Held
    with pytest.raises(AccelError, match="pages of 24"):
        dev.kv_cache(1, 4, 2, 24, 64, 3, 2)
    assert len(held) == 5 and not any(b.ptr for b in held)

    def short(shape, dtype):
        if len(held) == 3:
            raise AccelError(accel_amd.E_NO_DEVICE, "out of memory")
        return Held(shape, dtype)

    held.clear()
    dev.alloc = short
    with pytest.raises(AccelError, match="out of memory"):
        dev.kv_cache(1, 4, 2, 16, 64, 3, 2)
    assert len(held) == 3 and not any(b.ptr for b in held)
