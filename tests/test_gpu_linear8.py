"""linear8: what its backward pass makes, keeps and says, and autocast."""
import contextlib
import ctypes

import pytest
import torch
import torch.nn.utils.parametrize

import nano_nccl_b200 as nn
from nano_nccl_b200 import _lib, ops
from nano_nccl_b200.models import TinyGPT2

pytestmark = pytest.mark.gpu


@contextlib.contextmanager
def replaced(name, prototype, f):
    """Calls of the operators reach f(original, *arguments) instead of the C interface's `name`."""
    lib, native = nn.load(), nn.load_native_calls()
    address = {n: ctypes.cast(getattr(lib, n), ctypes.c_void_p).value for n in _lib._TRAIN}
    original = prototype(address[name])
    fake = prototype(lambda *arguments: f(original, *arguments))
    native.bind_train(nn.B200CclError, tuple(ctypes.cast(fake, ctypes.c_void_p).value if n == name else address[n] for n in _lib._TRAIN))
    try:
        yield
    finally:
        native.bind_train(nn.B200CclError, tuple(address[n] for n in _lib._TRAIN))


WEIGHT_GRAD = ctypes.CFUNCTYPE(ctypes.c_int, ctypes.c_void_p, ctypes.c_void_p)


def test_weight_gradients_are_made_for_who_asks():
    calls = []

    def count(original, *arguments):
        calls.append(1)
        return original(*arguments)

    x, w, b = (torch.randn(s, device="cuda", requires_grad=True) for s in ((40, 64), (32, 64), (32,)))
    dy = torch.randn(40, 32, device="cuda")
    with replaced("b2_weight_grad8", WEIGHT_GRAD, count):
        for wanted, expected in (((x,), 0), ((x, w), 1), ((w,), 1), ((x, w, b), 1)):
            y = ops.linear8(x, w, b)
            calls.clear()
            grads = torch.autograd.grad(y, wanted, dy)
            assert len(calls) == expected, wanted
            if wanted[0] is x:
                assert torch.equal(grads[0], dy @ w)


def test_a_weight_that_no_gradient_reads_may_change():
    """As behind torch's own projection: without a gradient of x, nothing reads the weight again."""
    for linear in (torch.nn.functional.linear, ops.linear8):
        x, w, dy = torch.randn(40, 64, device="cuda"), torch.randn(32, 64, device="cuda", requires_grad=True), torch.randn(40, 32, device="cuda")
        y = linear(x, w)
        with torch.no_grad():
            w.mul_(2.0)
        (dw,) = torch.autograd.grad(y, w, dy)
        assert torch.allclose(dw, dy.t() @ ops.unpack8(ops.pack8(x)), rtol=0.05, atol=0.5)
        y = linear(x.requires_grad_(), w)
        with torch.no_grad():
            w.mul_(2.0)
        with pytest.raises(RuntimeError, match="inplace"):
            torch.autograd.grad(y, x, dy)


def test_autocast_casts_as_torch_does():
    """A weight once in a context; 64-bit tensors, which torch leaves alone, not at all."""
    x, w, b = (torch.randn(s, device="cuda", requires_grad=True) for s in ((40, 64), (32, 64), (32,)))
    with torch.autocast("cuda", dtype=torch.bfloat16):
        first, second = ops.linear8(x, w, b), ops.linear8(x, w, b)
        assert first.grad_fn.next_functions[1][0] is second.grad_fn.next_functions[1][0]
        assert torch.equal(first, torch.nn.functional.linear(x, w, b)) and first.dtype == torch.bfloat16
        with pytest.raises(ValueError, match="Double"):
            ops.linear8(x.double(), w.double(), b.double())
        with torch.autocast("cuda", enabled=False):
            assert ops.linear8(x, w, b).dtype == torch.float32
    (first.float().sum() + second.float().sum()).backward()
    assert torch.equal(b.grad, torch.full_like(b, 80.0)) and w.grad.dtype == x.grad.dtype == torch.float32
    with torch.autocast("cuda", dtype=torch.float16), torch.no_grad():
        assert torch.equal(ops.linear8(x, w, b), torch.nn.functional.linear(x, w, b))


def test_a_failure_in_a_backward_pass_is_this_library_s_error():
    """The failing call is a stand-in on the host."""
    x, w = (torch.randn(s, device="cuda", requires_grad=True) for s in ((40, 64), (32, 64)))
    dy = torch.randn(40, 32, device="cuda")
    with replaced("b2_weight_grad8", WEIGHT_GRAD, lambda original, *arguments: 1):
        with pytest.raises(nn.B200CclError):
            ops.weight_grad8(dy, ops.pack8(x))
        for _ in range(2):
            y = ops.linear8(x, w)
            with pytest.raises(nn.B200CclError):
                y.backward(dy)
    with replaced("b2_weight_grad8", WEIGHT_GRAD, lambda original, *arguments: 2):
        with pytest.raises(ValueError):
            ops.linear8(x, w).backward(dy)
    ops.linear8(x, w).backward(dy)
    assert torch.equal(w.grad, ops.weight_grad8(dy, ops.pack8(x))[0])


def test_hooks_of_a_model_s_modules_are_called():
    """What is kept for the backward pass does not change which modules a forward pass goes through."""
    tokens = torch.zeros(1, 4, dtype=torch.long, device="cuda")
    names = {}
    for checkpoints in (None, "int8"):
        model = TinyGPT2(vocab=32, context=8, hidden=32, layers=1, heads=2, positions="rotary", checkpoints=checkpoints).cuda()
        seen = []
        for name, module in model.named_modules():
            module.register_forward_hook(lambda module, inputs, output, name=name: seen.append(name))
        model(tokens)
        names[checkpoints] = seen
        # A hook's result is what goes on, and a weight that is computed is the one that is used.
        model.blocks[0].mlp[2].register_forward_hook(lambda module, inputs, output: output * 0.0)
        torch.nn.utils.parametrize.register_parametrization(model.blocks[0].attn.c_proj, "weight", torch.nn.Identity())
        x = torch.randn(1, 4, 32, device="cuda")
        block = model.blocks[0]
        assert torch.equal(block(x), x + block.attn(block.ln_1(x)))
    assert names[None] == names["int8"] and "blocks.0.mlp.1" in names["int8"]


def test_head_norms_keep_8_bits_only_where_they_are_told_to():
    q, w, dy = (torch.randn(s, device="cuda") for s in ((9, 4, 64), (64,), (9, 4, 64)))
    q, w, p, f = q.requires_grad_(), w.requires_grad_(), torch.arange(9, device="cuda"), ops.rotary_frequencies(64)[0]
    given, full, short = (torch.autograd.grad(ops.qk_norm_rotary(q, None, w, None, p, f, **keep)[0], (q, w), dy) for keep in ({}, {"keep": None}, {"keep": "int8"}))
    assert all(torch.equal(a, b) for a, b in zip(given, full)) and not torch.equal(given[0], short[0])


def test_a_capture_inside_one_autocast_context_sees_later_weights():
    """Eager steps and the capture share the context, and so its cache of cast weights, which is not for a graph."""
    x, w = torch.randn(40, 64, device="cuda"), torch.randn(32, 64, device="cuda", requires_grad=True)
    with torch.autocast("cuda", dtype=torch.bfloat16):
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side), torch.no_grad():
            ops.linear8(x, w)
            eager = ops.linear8(x, w)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.no_grad(), torch.cuda.graph(graph):
            captured = ops.linear8(x, w)
        graph.replay()
        assert torch.equal(captured, eager)
        with torch.no_grad():
            w.mul_(2.0)
        graph.replay()
        assert torch.equal(captured, eager * 2)
    with torch.autocast("cuda", dtype=torch.bfloat16):  # a weight that was cast without a gradient has one all the same
        with torch.no_grad():
            ops.linear8(x, w)
        (dw,) = torch.autograd.grad(ops.linear8(x, w).float().sum(), w)
    assert dw.dtype == torch.float32 and dw.any()
