"""Bounded waits inside the weight gradient: with no time at all they run out, and the call's own results say so."""
import ctypes

import pytest
import torch

import nano_nccl_b200 as nn
from nano_nccl_b200 import ops
from test_cpu_train_ops import WeightGrad

pytestmark = pytest.mark.gpu

CODES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}


def prepared(dy, packed, bias):
    """(arguments of the C interface, gradients, what has to stay alive)"""
    tokens, outputs, inputs = dy.shape[0], dy.shape[1], packed.shape[1]
    dw, db = torch.zeros(outputs, inputs, dtype=dy.dtype, device="cuda"), torch.zeros(outputs, dtype=dy.dtype, device="cuda") if bias else None
    codes = packed.data.data_ptr()
    c = WeightGrad(dy.data_ptr(), dy.stride(0), tokens, outputs, inputs, CODES[dy.dtype], codes, codes + tokens * (-(-inputs // 32) * 32), dw.data_ptr(),
                   db.data_ptr() if bias else None, None)
    size = ctypes.c_size_t()
    assert nn.load().b2_weight_grad8_workspace(ctypes.byref(c), ctypes.byref(size)) == 0
    workspace = torch.empty(size.value, dtype=torch.uint8, device="cuda")
    c.workspace = workspace.data_ptr() if size.value else None
    return c, dw, db, (workspace, dy, packed)


def call(c, wait_ns):
    stream = ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)
    return nn.load().b2_weight_grad8_within(ctypes.byref(c), ctypes.c_ulonglong(wait_ns), stream)


# Every pair of CTAs waits for at least 200 steps of 64 tokens before it writes: far longer than the few polls that a wait always makes. Tiles of 512 outputs, whole and cut;
# one tile that all pairs share; the bias's gradient by the way and by a kernel of its own.
CASES = [(16384, 4096, 4096, torch.bfloat16, True), (1000003, 256, 250, torch.bfloat16, True), (1000003, 256, 250, torch.float16, False), (60000, 32, 18944, torch.float16, True)]


@pytest.mark.parametrize("tokens,inputs,outputs,dtype,bias", CASES)
def test_a_wait_that_runs_out_leaves_nan(tokens, inputs, outputs, dtype, bias):
    dy, packed = torch.ones(tokens, outputs, dtype=dtype, device="cuda") * 2.0 ** -10, ops.pack8(torch.ones(tokens, inputs, dtype=dtype, device="cuda"))
    want = ops.weight_grad8(dy, packed, bias=bias)
    torch.cuda.synchronize()
    ops.check_async_error()
    c, dw, db, _ = prepared(dy, packed, bias)
    assert call(c, 0) == 0
    torch.cuda.synchronize()
    assert dw.isnan().all() and (db is None or db.isnan().all())
    # Nobody else is told: the next call works, and asking says it once.
    again = ops.weight_grad8(dy, packed, bias=bias)
    assert torch.equal(again[0], want[0]) and (not bias or torch.equal(again[1], want[1]))
    with pytest.raises(nn.B200CclError, match="ran out"):
        ops.check_async_error()
    ops.check_async_error()
    assert call(c, 2 * 10 ** 9) == 0
    torch.cuda.synchronize()
    assert torch.equal(dw, want[0]) and (db is None or torch.equal(db, want[1]))
    ops.check_async_error(0)


def test_a_replayed_call_says_so_too():
    dy, packed = torch.ones(1000003, 256, dtype=torch.bfloat16, device="cuda"), ops.pack8(torch.ones(1000003, 256, dtype=torch.bfloat16, device="cuda"))
    c, dw, db, _ = prepared(dy, packed, True)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        assert call(c, 0) == 0
    for _ in range(2):
        dw.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert dw.isnan().all() and db.isnan().all()
        with pytest.raises(nn.B200CclError, match="ran out"):
            ops.check_async_error(torch.device("cuda", 0))
