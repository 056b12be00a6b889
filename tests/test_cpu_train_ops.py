"""Training operators without a GPU: what they refuse, through Python and through the C interface, and the model that calls them."""
import ctypes
import math

import pytest
import torch

import nano_nccl_b200 as nn
from nano_nccl_b200 import ops
from nano_nccl_b200.models import TinyGPT2


@pytest.fixture(scope="module")
def lib(native_build):
    return nn.load()


def test_cpu_tensors_and_wrong_arguments_are_refused(lib):
    x, p, f = torch.ones(4, 3, 64), torch.arange(4), torch.ones(32, dtype=torch.float64)
    packed = ops.Packed8(torch.zeros(4 * 3 * 66, dtype=torch.uint8), (4, 3, 64), torch.float32)
    for call in (lambda: ops.pack8(x), lambda: ops.unpack8(packed), lambda: ops.unpack8(x), lambda: ops.gelu8(x), lambda: ops.gelu8(x, "sigmoid"),
                 lambda: ops.linear8(x, torch.ones(8, 64)), lambda: ops.weight_grad8(x, packed), lambda: ops.weight_grad8(x, x),
                 lambda: ops.weight_grad8(x[:2], packed), lambda: ops.weight_grad8(x.half(), packed), lambda: ops.rotary(x, None, p, f),
                 lambda: ops.rotary(None, None, p, f), lambda: ops.rotary(x, None, p, f, layout="thirds"), lambda: ops.pack8("x"),
                 lambda: ops.qk_norm_rotary(x, None, torch.ones(64), None, p, f), lambda: ops.qk_norm_rotary(x, x, None, None, p, f, keep="int4"),
                 lambda: ops.qk_norm_rotary(x, x, None, None, p, f, eps=float("nan"))):
        with pytest.raises(ValueError):
            call()


def test_frequencies():
    with pytest.raises(ValueError):
        ops.rotary_frequencies(63, device="cpu")
    for kw in (dict(scaling="dynamic"), dict(scaling="yarn", factor=2.0), dict(factor=0.5), dict(base=1.0), dict(scaling="yarn", context=64, fast=1.0, slow=2.0)):
        with pytest.raises(ValueError):
            ops.rotary_frequencies(64, device="cpu", **kw)
    with pytest.raises(ValueError):
        ops.rotary_frequencies(2, scaling="ntk", factor=2.0, device="cpu")
    f, m = ops.rotary_frequencies(8, base=16.0, device="cpu")
    assert f.dtype == torch.float64 and m == 1.0 and torch.allclose(f, torch.tensor([1.0, 0.5, 0.25, 0.125], dtype=torch.float64))
    # yarn at its ends: pairs of more than `fast` turns stay, those of fewer than `slow` are divided, and the magnitude grows with the factor
    f, m = ops.rotary_frequencies(128, scaling="yarn", factor=16.0, context=2048, device="cpu")
    plain = 10000.0 ** (-torch.arange(64, dtype=torch.float64) / 64)
    assert torch.equal(f[:10], plain[:10]) and torch.allclose(f[-5:], plain[-5:] / 16) and m == pytest.approx(0.1 * math.log(16.0) + 1)
    # ... where no pair makes fewer than `slow` turns (none is divided in full), and where none makes as many (all are)
    f, _ = ops.rotary_frequencies(64, scaling="yarn", factor=16.0, context=131072, device="cpu")
    plain = 10000.0 ** (-torch.arange(32, dtype=torch.float64) / 32)
    assert (plain * 131072 / (2 * math.pi) > 1).all() and (f > plain / 16 * 1.01).all()
    f, _ = ops.rotary_frequencies(64, scaling="yarn", factor=16.0, context=4, device="cpu")
    assert torch.allclose(f, plain / 16, rtol=1e-14, atol=0)


class Heads(ctypes.Structure):
    _fields_ = [("heads", ctypes.c_int), ("x", ctypes.c_void_p), ("x_strides", ctypes.c_longlong * 3), ("grad", ctypes.c_void_p),
                ("grad_strides", ctypes.c_longlong * 3), ("out", ctypes.c_void_p), ("weight", ctypes.c_void_p), ("codes", ctypes.c_void_p),
                ("scales", ctypes.c_void_p), ("weight_grad", ctypes.c_void_p), ("partial", ctypes.c_void_p)]


class Rotation(ctypes.Structure):
    _fields_ = [("dtype", ctypes.c_int), ("batch", ctypes.c_longlong), ("tokens", ctypes.c_longlong), ("dim", ctypes.c_int), ("rotated", ctypes.c_int),
                ("interleaved", ctypes.c_int), ("inverse", ctypes.c_int), ("norm", ctypes.c_int), ("eps", ctypes.c_float), ("magnitude", ctypes.c_float),
                ("positions", ctypes.c_void_p), ("position_bytes", ctypes.c_int), ("position_strides", ctypes.c_longlong * 2),
                ("frequencies", ctypes.c_void_p), ("side", Heads * 2)]


class WeightGrad(ctypes.Structure):
    _fields_ = [("dy", ctypes.c_void_p), ("stride", ctypes.c_longlong), ("tokens", ctypes.c_size_t), ("outputs", ctypes.c_size_t),
                ("inputs", ctypes.c_size_t), ("dtype", ctypes.c_int), ("codes", ctypes.c_void_p), ("scales", ctypes.c_void_p),
                ("weight_grad", ctypes.c_void_p), ("bias_grad", ctypes.c_void_p), ("workspace", ctypes.c_void_p)]


def refused(lib, code, words):
    assert code == 2, lib.b2_last_error()
    assert words in lib.b2_last_error().decode()


def test_c_interface_refuses_what_would_leave_its_buffers(lib):
    P, LL, S, I = ctypes.c_void_p, ctypes.c_longlong, ctypes.c_size_t, ctypes.c_int
    pack = lambda x, rows, columns, dtype, codes, scales: lib.b2_pack8(P(x), LL(columns), S(rows), S(columns), I(dtype), P(codes), P(scales), None)  # noqa: E731
    refused(lib, pack(4096, 2, 64, 3, 4096, 4096), "dtype")
    refused(lib, pack(None, 2, 64, 0, 4096, 4096), "non-null")
    refused(lib, pack(4096, 2, 64, 0, None, 4096), "non-null")
    refused(lib, pack(4096, 2, 64, 0, 4100, 4096), "32 bytes")
    refused(lib, pack(4097, 2, 64, 1, 4096, 4096), "aligned to its elements")
    refused(lib, pack(4096, 1 << 26, 1 << 10, 0, 4096, 4096), "2^30")
    refused(lib, lib.b2_unpack8(P(4096), P(4096), S(2), S(64), I(0), None, None), "non-null")
    refused(lib, lib.b2_gelu8_forward(P(4096), LL(64), S(2), S(64), I(0), I(0), None, None, None, None), "non-null")
    refused(lib, lib.b2_gelu8_backward(P(4096), LL(64), None, P(4096), S(2), S(64), I(0), I(0), P(4096), None), "non-null")
    assert pack(None, 0, 64, 0, None, None) == 0  # nothing to do

    w = WeightGrad(4096, 64, 32, 64, 64, 2, 4096, 4096, 4096, None, 4100)
    refused(lib, lib.b2_weight_grad8(ctypes.byref(w), None), "workspace")
    w.workspace, w.dtype = 4096, 7
    refused(lib, lib.b2_weight_grad8(ctypes.byref(w), None), "dtype")
    w.dtype, w.codes = 2, 4098
    refused(lib, lib.b2_weight_grad8(ctypes.byref(w), None), "32 bytes")
    w.codes, w.weight_grad = 4096, None
    refused(lib, lib.b2_weight_grad8(ctypes.byref(w), None), "weight_grad")
    refused(lib, lib.b2_weight_grad8(None, None), "null")

    def rotation(**kw):
        side = Heads(heads=4, x=4096, x_strides=(LL * 3)(0, 256, 64), out=4096)
        r = Rotation(dtype=2, batch=1, tokens=8, dim=64, rotated=64, magnitude=1.0, positions=4096, position_bytes=8, frequencies=4096)
        r.side[0] = side
        for k, v in kw.items():
            setattr(r.side[0] if k in dict(Heads._fields_) else r, k, v)
        return ctypes.byref(r)

    for words, kw in (("even", dict(dim=63)), ("even", dict(dim=258)), ("rotated", dict(rotated=66)), ("rotated", dict(rotated=31)),
                      ("2^31", dict(tokens=1 << 31)), ("4 or 8", dict(position_bytes=2)), ("positions", dict(positions=None)),
                      ("neither", dict(heads=0)), ("65536", dict(heads=1 << 16)), ("non-null", dict(x=None)), ("aligned", dict(out=4097)),
                      ("weight", dict(norm=1))):
        refused(lib, lib.b2_rotate_heads(rotation(**kw), None), words)
    for words, kw in (("weight", {}), ("grad", dict(weight=4096)), ("partial", dict(weight=4096, grad=4096))):
        refused(lib, lib.b2_rotate_heads_backward(rotation(**kw), None), words)


def test_model_options():
    torch.manual_seed(0)
    plain = TinyGPT2(vocab=32, context=8, hidden=32, layers=1, heads=2)
    assert "blocks.0.attn.in_proj_weight" in plain.state_dict() and "wpe.weight" in plain.state_dict()
    assert plain(torch.zeros(1, 8, dtype=torch.long)).shape == (1, 8, 32)
    assert TinyGPT2(vocab=32, context=8, hidden=6, layers=1, heads=2)(torch.zeros(1, 8, dtype=torch.long)).shape == (1, 8, 32)  # heads of 3
    model = TinyGPT2(vocab=32, context=8, hidden=32, layers=1, heads=2, positions="rotary", qk_norm=True, checkpoints="int8")
    names = model.state_dict()
    assert "wpe.weight" not in names and "blocks.0.attn.q_norm" in names and {n for n in names if ".mlp." in n} == {n for n in plain.state_dict() if ".mlp." in n}
    with pytest.raises(ValueError):
        model(torch.zeros(1, 8, dtype=torch.long))  # these operators have no CPU form
    for kw in (dict(positions="sine"), dict(checkpoints="fp8"), dict(hidden=6, heads=2, positions="rotary"), dict(hidden=32, heads=3, qk_norm=True)):
        with pytest.raises(ValueError):
            TinyGPT2(**kw)
