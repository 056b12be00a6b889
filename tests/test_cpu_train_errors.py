"""What the training operators say of failures, without a GPU."""
import ctypes

import pytest

import nano_nccl_b200 as nn
from nano_nccl_b200 import ops


@pytest.fixture(scope="module")
def lib(native_build):
    return nn.load()


def test_asking_for_waits_that_ran_out(lib):
    ops.check_async_error(0)  # no call so far
    ops.check_async_error("cuda:5")
    with pytest.raises(ValueError, match="no such device"):
        ops.check_async_error(-1)
    assert lib.b2_weight_grad8_within(None, ctypes.c_ulonglong(5), None) == 2 and b"null" in lib.b2_last_error()


def test_fake_tensors_are_refused(lib):
    import torch
    from torch._subclasses.fake_tensor import FakeTensorMode
    with FakeTensorMode() as mode:
        x, f, p = torch.empty(5, 2, 64, device="cuda"), torch.empty(32, dtype=torch.float64, device="cuda"), torch.empty(5, dtype=torch.int64, device="cuda")
    calls = [lambda: ops.pack8(x), lambda: ops.gelu8(x), lambda: ops.linear8(x, x[0]), lambda: ops.rotary(x, None, p, f), lambda: ops.qk_norm_rotary(x, x, x[0, 0], x[0, 0], p, f)]
    for call in calls:
        with pytest.raises(ValueError, match="memory of its own"):
            call()
        with mode, pytest.raises(ValueError, match="traced"):
            call()


def test_a_model_of_heads_that_do_not_fit_is_refused_when_it_is_made():
    from nano_nccl_b200.models import TinyGPT2
    for options in ({}, {"checkpoints": "int8"}, {"positions": "rotary"}):
        with pytest.raises((ValueError, AssertionError)):
            TinyGPT2(hidden=32, heads=3, **options)
    TinyGPT2(hidden=32, heads=4, checkpoints="int8")
