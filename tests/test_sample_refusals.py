"""Logits that start between two numbers of their type are refused (CPU: the check runs
before a device is touched)."""
import pytest

from accel_amd import BF16, F16, F32
from test_draft_refusals import sample
from test_kv_refusals import A, refused, tensor


@pytest.mark.parametrize("dtype,off", [(F32, 1), (F32, 2), (F32, 3), (F16, 1), (BF16, 3)])
def test_logits_between_two_numbers(dtype, off):
    refused(sample(x=tensor((5, 100), dtype, A + off)), "Sample", "aligned")


@pytest.mark.parametrize("dtype,off", [(F32, 4), (F32, 12), (F16, 2), (BF16, 6)])
def test_logits_at_any_number(dtype, off):
    # what is refused is what comes after the logits
    refused(sample(x=tensor((5, 100), dtype, A + off), u=None), "random numbers")
