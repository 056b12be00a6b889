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
