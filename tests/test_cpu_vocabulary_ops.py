"""The operators over a vocabulary without a GPU: what they refuse, through Python and through the C interface, and the model that calls them."""
import ctypes

import pytest
import torch

import nano_nccl_b200 as nn
from nano_nccl_b200 import ops
from nano_nccl_b200.models import TinyGPT2


@pytest.fixture(scope="module")
def lib(native_build):
    return nn.load()


def test_cpu_tensors_and_wrong_arguments_are_refused(lib):
    x, w, t = torch.ones(4, 64), torch.ones(10, 64), torch.zeros(4, dtype=torch.int64)
    entries = torch.zeros(4, 3, dtype=torch.int64)
    for call in (lambda: ops.embedding(t, w), lambda: ops.embedding("x", w), lambda: ops.linear_cross_entropy(x, w, t), lambda: ops.linear_cross_entropy(x, w, t, reduction="median"),
                 lambda: ops.linear_distillation(x, w, torch.ones(4, 3), entries), lambda: ops.linear_distillation(x, w, torch.ones(4, 3), entries, reduction="batchmean"),
                 *(lambda v=v: ops.linear_distillation(x, w, torch.ones(4, 3), entries, temperature=v) for v in (0.0, -1.0, float("inf"), float("nan")))):
        with pytest.raises(ValueError):
            call()


def test_fake_tensors_are_refused(lib):
    from torch._subclasses.fake_tensor import FakeTensorMode
    with FakeTensorMode() as mode:
        x, t = torch.empty(5, 64, device="cuda"), torch.empty(5, dtype=torch.int64, device="cuda")
    for call in (lambda: ops.embedding(t, x), lambda: ops.linear_cross_entropy(x, x, t), lambda: ops.linear_distillation(x, x, x[:, :3], t[:, None].expand(5, 3))):
        with pytest.raises(ValueError, match="memory of its own"):
            call()
        with mode, pytest.raises(ValueError, match="traced"):
            call()


P, LL, S, I, F = ctypes.c_void_p, ctypes.c_longlong, ctypes.c_size_t, ctypes.c_int, ctypes.c_float


class Embedding(ctypes.Structure):
    _fields_ = [("dtype", I), ("tokens", P), ("token_bytes", I), ("token_stride", LL), ("count", S), ("vocabulary", S), ("width", S), ("scale", F), ("rows", P),
                ("stride", LL), ("out", P), ("workspace", P)]


class VocabularyLoss(ctypes.Structure):
    _fields_ = [("dtype", I), ("x", P), ("x_stride", LL), ("weight", P), ("weight_stride", LL), ("tokens", S), ("width", S), ("vocabulary", S), ("targets", P),
                ("target_bytes", I), ("target_strides", LL * 2), ("entries", I), ("teacher", P), ("teacher_dtype", I), ("teacher_strides", LL * 2), ("temperature", F),
                ("reduction", I), ("loss", P), ("kept", P), ("loss_grad", P), ("loss_grad_stride", LL), ("x_grad", P), ("weight_grad", P), ("workspace", P)]


def refused(lib, code, words):
    assert code == 2, lib.b2_last_error()
    assert words in lib.b2_last_error().decode()


def test_c_interface_refuses_what_would_leave_its_buffers(lib):
    def embedding(**kw):
        e = Embedding(dtype=2, tokens=4096, token_bytes=8, token_stride=1, count=4, vocabulary=10, width=64, scale=1.0, rows=4096, stride=64, out=4096, workspace=4096)
        for k, v in kw.items():
            setattr(e, k, v)
        return ctypes.byref(e)

    refused(lib, lib.b2_embed(None, None), "null")
    for words, kw in (("dtype", dict(dtype=3)), ("4 or 8", dict(token_bytes=2)), ("at least one", dict(vocabulary=0)), ("at least one", dict(width=0)),
                      ("too many", dict(vocabulary=1 << 31)), ("non-null", dict(tokens=None)), ("non-null", dict(rows=None)), ("non-null", dict(out=None)),
                      ("aligned", dict(tokens=4100)), ("aligned", dict(rows=4097)), ("aligned", dict(out=4097))):
        refused(lib, lib.b2_embed(embedding(**kw), None), words)
    for words, kw in (("too many", dict(count=1 << 30)), ("workspace", dict(workspace=None)), ("workspace", dict(workspace=4100)), ("16 bytes", dict(out=4098)), ("non-null", dict(out=None, count=0))):
        refused(lib, lib.b2_embed_backward(embedding(**kw), None), words)
    size = S()
    refused(lib, lib.b2_embed_backward_workspace(embedding(), None), "non-null")
    assert lib.b2_embed_backward_workspace(embedding(workspace=None, out=None), ctypes.byref(size)) == 0 and size.value > 0
    assert lib.b2_embed(embedding(count=0, tokens=None, rows=None, out=None), None) == 0  # nothing to do

    def loss(**kw):
        c = VocabularyLoss(dtype=2, x=4096, x_stride=64, weight=4096, weight_stride=64, tokens=4, width=64, vocabulary=10, targets=4096, target_bytes=8,
                           target_strides=(LL * 2)(1, 1), temperature=1.0, loss=4096, kept=4096, loss_grad=4096, loss_grad_stride=1, x_grad=4096, weight_grad=4096, workspace=4096)
        for k, v in kw.items():
            setattr(c, k, v)
        return ctypes.byref(c)

    both = [("null", None)] + [(words, loss(**kw)) for words, kw in (
        ("dtype", dict(dtype=-1)), ("at least one", dict(vocabulary=0)), ("at least one", dict(width=0)), ("too many", dict(tokens=1 << 30)), ("too many", dict(vocabulary=1 << 30)),
        ("4 or 8", dict(target_bytes=1)), ("reduction", dict(reduction=3)), ("256", dict(entries=257)), ("256", dict(entries=-1)), ("temperature", dict(entries=2, teacher=4096, temperature=0.0)),
        ("temperature", dict(entries=2, teacher=4096, temperature=float("nan"))), ("no temperature", dict(temperature=2.0)), ("non-null", dict(x=None)), ("non-null", dict(weight=None)),
        ("non-null", dict(targets=None)), ("non-null", dict(kept=None)), ("aligned", dict(x=4097)), ("aligned", dict(targets=4100)), ("backwards", dict(x_stride=-64)),
        ("backwards", dict(weight_stride=-64)), ("workspace", dict(workspace=None)), ("workspace", dict(workspace=4100)))]
    for words, call in both:
        refused(lib, lib.b2_vocabulary_loss_forward(call, None), words)
        refused(lib, lib.b2_vocabulary_loss_backward(call, None), words)
    for words, kw in (("loss", dict(loss=None)), ("aligned", dict(loss=4098)), ("teacher", dict(entries=2)), ("dtype", dict(entries=2, teacher=4096, teacher_dtype=5))):
        refused(lib, lib.b2_vocabulary_loss_forward(loss(**kw), None), words)
    for words, kw in (("loss_grad", dict(loss_grad=None)), ("loss_grad", dict(loss_grad=4098)), ("aligned", dict(x_grad=4097)), ("aligned", dict(weight_grad=4097))):
        refused(lib, lib.b2_vocabulary_loss_backward(loss(**kw), None), words)
    assert lib.b2_vocabulary_loss_forward(loss(tokens=0, x=None, targets=None, kept=None, loss=None, workspace=None), None) == 0  # nothing to do
    # Gradients with the loss: of bf16, of one loss for all rows, of large products, and where they are wanted; otherwise no bytes are asked for, and the call is refused.
    large = dict(tokens=4096, vocabulary=50000, width=768, x_stride=768, weight_stride=768, reduction=1)
    for kw in (dict(reduction=1), {**large, "dtype": 0}, {**large, "dtype": 1}, {**large, "reduction": 0}, {**large, "x_grad": None, "weight_grad": None}):
        assert lib.b2_vocabulary_loss_both_workspace(loss(**kw), ctypes.byref(size)) == 0 and size.value == 0
        refused(lib, lib.b2_vocabulary_loss_both(loss(**kw), None), "at once")
    refused(lib, lib.b2_vocabulary_loss_both_workspace(loss(**large), None), "non-null")
    for words, kw in (("loss must be", dict(loss=None)), ("workspace", dict(workspace=None)), ("aligned", dict(x_grad=4097)), ("aligned", dict(loss=4098))):
        refused(lib, lib.b2_vocabulary_loss_both(loss(**{**large, **kw}), None), words)
    for words, kw in (("bf16", dict(dtype=0)), ("loss_grad", dict(loss_grad=None)), ("aligned", dict(weight_grad=4097))):
        refused(lib, lib.b2_vocabulary_loss_times(loss(**kw), None), words)
    assert lib.b2_vocabulary_loss_times(loss(x_grad=None, weight_grad=None), None) == 0  # nothing to do
    refused(lib, lib.b2_vocabulary_loss_within(loss(), 3, ctypes.c_ulonglong(1), None), "pass")
    refused(lib, lib.b2_vocabulary_loss_check_async_error(-1), "device")


def test_asking_for_waits_that_ran_out(lib):
    ops.check_async_error(0)  # no call so far
    with pytest.raises(ValueError, match="no such device"):
        ops.check_async_error(-1)


def test_model_options():
    torch.manual_seed(0)
    tokens, targets = torch.randint(0, 32, (2, 8)), torch.randint(0, 32, (2, 8))
    targets[0, 5:] = -1
    plain = TinyGPT2(vocab=32, context=8, hidden=32, layers=1, heads=2)
    loss = plain(tokens, targets)
    logits = plain(tokens)
    assert torch.allclose(loss, torch.nn.functional.cross_entropy(logits[targets >= 0], targets[targets >= 0]), rtol=1e-6)
    assert plain(tokens, torch.full_like(targets, -5)) == 0
    fused = TinyGPT2(vocab=32, context=8, hidden=32, layers=1, heads=2, vocabulary="fused")
    assert fused.state_dict().keys() == plain.state_dict().keys()
    with pytest.raises(ValueError):
        fused(tokens)  # these operators have no CPU form
    with pytest.raises(ValueError, match="fused"):
        plain(tokens, teacher=(torch.ones(2, 8, 3), torch.zeros(2, 8, 3, dtype=torch.long)))
    with pytest.raises(ValueError, match="not both"):
        fused(tokens, targets, teacher=(1, 2))
    with pytest.raises(ValueError):
        TinyGPT2(vocabulary="sparse")
