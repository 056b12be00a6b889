"""The two ends of a training step over a vocabulary: the lookup of tokens, and losses whose logits are never stored.

``weight`` is [vocabulary, width], the same matrix at both ends where a model ties them. Tokens and targets are int64 or int32, of any shape and strides. A negative one
stands for no token (the padding of a sequence): it is looked up as zeros, has no loss and no gradient, and does not count in a mean. One that is not below
the vocabulary makes NaN, so that a loss scaler sees it. (Rows that do not count still go through the products: their hidden states must be numbers, of any size.)

The logits of 8192 tokens over 50257 words take 1.6 GB in 32 bits, and their gradient as much again. The losses here make them tile by tile on the tensor cores
and keep a few numbers for each row; the backward pass makes them again, by pieces of the vocabulary, each of which is an operand of 16 bits (float32: two of them) of the two products that
make the gradients. It needs 512 MB at most for that, or 4096 words of the vocabulary.

bfloat16, with one loss for all rows and a product large enough: the logits are made once. A call whose inputs want gradients makes them with the loss, by pieces of the rows (1 GB of workspace,
and as much again at most for sums where there are several), and keeps them; the backward pass multiplies them by what comes back, which rounds once more unless that is a power of two.
Asked for a second time (``retain_graph``) they are made from the logits. A loss whose gradient nobody will ask for is cheaper under
``torch.no_grad()``; one of each row, added up by the caller, takes less memory, and makes its logits twice.

CUDA tensors of float32, float16 or bfloat16; calls run on the current stream of the tensors' device. As with the other operators of this package (:mod:`.checkpoint8`)
reverse-mode gradients are made once, and tracing, forward mode and ``torch.func`` are refused; a step captured into a CUDA graph is captured with
its backward pass and on one stream, after eager steps of the same parameters have been run and their graphs dropped.
"""
from .._lib import load_native_calls

_REDUCTIONS = {"none": 0, "mean": 1, "sum": 2}


def _reduction(name):
    if name not in _REDUCTIONS:
        raise ValueError(f"unknown reduction '{name}'")
    return _REDUCTIONS[name]


def embedding(tokens, weight, scale=1.0):
    """``scale * weight[tokens]``, of shape ``[*tokens.shape, width]``, rounded once.

    The weight's gradient is made by sorting the tokens: sums are held in 32 bits, in the order of the tokens, rounded once, and do not
    depend on timing; rows of words that do not occur are zeros."""
    return load_native_calls().embedding(tokens, weight, scale)


def linear_cross_entropy(x, weight, targets, reduction="mean"):
    """``torch.nn.functional.cross_entropy(x @ weight.T, targets)`` without the logits: the loss of each row, ``log sum exp(z) - z[target]``, or with ``reduction`` "mean" or "sum"
    one of all of them (a mean over the rows that have a target; 0 where none has). ``x``: [..., width], ``targets``: [...]. The loss is float32, gradients have the types of ``x``
    and ``weight``, which are the same. Under autocast both are cast as those of ``linear``.

    What the logits lose is what 32-bit sums lose; the gradient of the logits is rounded to the type of ``x`` before it is multiplied. float32: operands have 22 bits, or where that is
    more 2^-39 of the largest element of ``weight``, of the row of ``x`` (in the gradient of ``weight``: of the rows of ``x`` that count, times their weights in the loss), and of 1 in the softmax.
    float16, a loss of each row: the gradient of ``weight`` takes ``x`` times a power of two of its row's weight, exactly, down to 2^-28 of the largest such element."""
    return load_native_calls().linear_cross_entropy(x, weight, targets, _reduction(reduction))


def linear_distillation(x, weight, teacher_logits, teacher_tokens, temperature=1.0, reduction="mean"):
    """The divergence of a student, whose logits are ``x @ weight.T``, from a teacher of whose logits the largest were stored: for each row ``temperature ** 2 * sum p (log p - log q)``,
    ``p`` being the softmax of ``teacher_logits / temperature`` over the row's entries and ``q`` that of the student's logits / temperature over the vocabulary.

    ``teacher_logits`` (float32, float16 or bfloat16) and ``teacher_tokens``: [..., entries], 1 to 256 of them. An entry is left out where its token is negative or its
    logit -infinity; entries of the same token add up. No gradient is made of the teacher. The rest is as in :func:`linear_cross_entropy`."""
    if not 0.0 < float(temperature) < float("inf"):
        raise ValueError("the temperature must be positive")
    return load_native_calls().linear_distillation(x, weight, teacher_logits, teacher_tokens, temperature, _reduction(reduction))
