"""Activations kept in 8 bits for the backward pass.

What a training step keeps between forward and backward bounds the batch of a GPU, and with it the tokens that
one gradient all-reduce pays for. Here an activation is kept as blocks of 32 neighbouring elements of its last
axis: a power of two for the block and 8 bits for each element, 33 bytes instead of 64. With the block's largest
magnitude in ``[2^a, 2^(a+1))`` the step is ``2^q``, ``q = max(a - 6, -126)`` (-24 for fp16), and an element becomes

    x^ = sign(x) * min(round(|x| / 2^q), 127) * 2^q        (ties to even)

which is exact in the activation's own type. Forward results are made from the activation itself and do not change; gradients are
exactly those of the formula at ``x^``. A block that holds an infinity or NaN reads back as NaN, so that a loss scaler sees it.

CUDA tensors of float32, float16 or bfloat16; calls run on the current stream of the tensors' device. The kernels are this library's own, but for the result of
:func:`linear8` and the gradient of its input, which are torch's products.
A step captured into a CUDA graph is captured with its backward pass and on one stream, after eager steps of the same parameters have
been run and their graphs dropped, as for any torch module.

Unlike the collectives these are functions and no registered torch operators: reverse-mode gradients are made once, and tracing, fake tensors,
forward mode, ``torch.func`` and tensors that stand for others are refused. (``torch.compile`` leaves its graph for them.)
"""
import torch

from .._lib import B200CclError, load, load_native_calls

_APPROXIMATIONS = {"none": False, "tanh": True}


class Packed8:
    """An activation in 8 bits, from :func:`pack8`: ``data`` (bytes: the codes, rows padded to whole blocks, then one scale for each
    block), and the ``shape`` and ``dtype`` that it reads back as."""

    __slots__ = ("data", "shape", "dtype")

    def __init__(self, data, shape, dtype):
        self.data, self.shape, self.dtype = data, tuple(shape), dtype

    @property
    def nbytes(self):
        return self.data.numel()

    def __repr__(self):
        return f"Packed8(shape={self.shape}, dtype={self.dtype}, nbytes={self.nbytes})"


def _packed(what, p):
    if not isinstance(p, Packed8):
        raise ValueError(f"{what} must be a Packed8, as pack8() returns it")


def pack8(x):
    """``x`` (any shape with at least one axis, any strides) in 8 bits. No gradient flows through it."""
    return Packed8(load_native_calls().pack8(x), x.shape, x.dtype)


def unpack8(packed):
    """What :func:`pack8` kept, as a new tensor without gaps."""
    _packed("unpack8's argument", packed)
    return load_native_calls().unpack8(packed.data, packed.shape, packed.dtype)


def gelu8(x, approximate="none"):
    """``torch.nn.functional.gelu(x, approximate)``; the backward pass reads ``x`` in 8 bits, written in the same pass as the result.

    float32: within 4e-7 of the largest of 1 and the result; relative to results far out on the negative side 8e-6 up to -12 (tanh: 4e-5 until they
    vanish), where exp's argument is rounded."""
    if approximate not in _APPROXIMATIONS:
        raise ValueError(f"unknown approximation '{approximate}'")
    return load_native_calls().gelu8(x, _APPROXIMATIONS[approximate])


def weight_grad8(dy, packed, bias=False):
    """Gradients of a projection ``y = x @ w.T + b`` whose input was kept: ``(dw, db)``, ``db`` None unless ``bias``.

    ``dy``: [..., outputs], ``packed``: of [..., inputs] with the same leading axes and the same dtype. Sums over all leading axes are held in
    32 bits and rounded once to that dtype (float32: products of full 24-bit numbers); the tensor cores' additions cut instead of rounding, which in
    16-bit types takes 7e-5 of a long sum of one sign, 3e-4 at most, however long it is. Results do not depend on timing."""
    _packed("packed", packed)
    if isinstance(dy, torch.Tensor):
        if dy.dtype != packed.dtype:
            raise ValueError(f"dy has dtype {dy.dtype}, the packed input {packed.dtype}")
        if dy.shape[:-1] != packed.shape[:-1]:
            raise ValueError(f"dy of shape {tuple(dy.shape)} does not belong to an input of shape {packed.shape}")
    return load_native_calls().weight_grad8(dy, packed.data, packed.shape[-1], bias)


def linear8(x, weight, bias=None):
    """``torch.nn.functional.linear(x, weight, bias)``; the weight's gradient reads ``x`` in 8 bits (:func:`weight_grad8`).
    Under autocast its arguments are cast as those of ``linear``."""
    return load_native_calls().linear8(x, weight, bias)


def check_async_error(device=None):
    """Raises B200CclError if a bounded wait inside a weight gradient, or a loss over a vocabulary or its gradients (:mod:`.vocabulary`), on ``device`` (default: the
    current one) ran out since this was last called. Such results are NaN, so a loss scaler
    sees them too (gradients made with a loss may have been made again, and be right). Synchronize first: only calls that are done are known."""
    index = torch.cuda.current_device() if device is None else torch.device(device).index if not isinstance(device, int) else device
    index = torch.cuda.current_device() if index is None else index
    codes = []
    for what in (load().b2_train_check_async_error, load().b2_vocabulary_loss_check_async_error):
        codes.append(what(index))  # (both are asked, and forget, whatever the first says)
        if codes[-1] != 0:
            failure = load().b2_last_error()
    if any(codes):
        raise (ValueError if 2 in codes else B200CclError)(failure.decode("utf-8", "replace"))
