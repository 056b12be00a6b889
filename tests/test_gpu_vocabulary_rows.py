"""Losses over a vocabulary: what one row is must not reach another's loss or gradient, and the ways that a call may take are each held to what that way may lose."""

import pytest
import torch

import plain_vocabulary as plain
from test_gpu_vocabulary_loss import DTYPES, cross_entropy, distillation, gen, inputs, made_with_the_loss, run, teacher

pytestmark = pytest.mark.gpu


# ---- what comes back to rows that are weighted one by one ------------------------------------------------

@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("frozen", [False, True])
def test_a_weight_that_is_no_number_stays_in_its_row(dtype, frozen):
    x, w, t = inputs(80, 700, 72, dtype)
    t = t.clamp(min=0)
    dloss = torch.rand(80, device="cuda", generator=gen(5)) + 0.5
    spoilt, without = dloss.clone(), dloss.clone()
    spoilt[5], spoilt[9], spoilt[70] = float("inf"), float("nan"), -float("inf")
    without[[5, 9, 70]] = 0.0
    logits, tokens = teacher(80, 5, 700, dtype)
    others = without != 0.0
    for call in (cross_entropy(t, "none"), distillation(logits, tokens, 2.0, "none")):
        def gradients(back):
            a, b = x.clone().requires_grad_(), w.clone().requires_grad_(not frozen)
            return torch.autograd.grad(call(a, b), (a,) if frozen else (a, b), back)
        got, want = gradients(spoilt), gradients(without)
        assert torch.equal(got[0][others], want[0][others]) and want[0].isfinite().all()
        assert not got[0][~others].isfinite().any()
        if not frozen:
            assert not got[1].isfinite().any() and want[1].isfinite().all()


# ---- which way a call takes, and what it may lose there --------------------------------------------------

def loses_its_own_rounding(out, want, dtype, what=""):
    for name in ("dx", "dw"):
        exact = want[name][0]
        rounded = (exact.to(dtype).double() - exact).norm()
        # P in two parts is off by 2^-16 at most, the softmax by what its logits are: with at most 4096 products of about 0.03 that may lose 2^-23 of themselves 256 times, 1e-5, beside roundings of
        # at least 2^-13 in the mean.
        assert (out[name].double() - exact).norm() <= 1.1 * rounded + 1e-30, f"{what} {name}"


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("rows,vocabulary,width", [(1, 152064, 1024), (12, 152064, 1024), (64, 262144, 512)])
def test_gradients_of_few_rows_over_a_large_vocabulary(dtype, rows, vocabulary, width):
    x, w, t = inputs(rows, vocabulary, width, dtype)
    dloss = torch.randn(rows, device="cuda", generator=gen(9))
    out = run(cross_entropy(t, "none"), x, w, dloss)
    loses_its_own_rounding(out, plain.losses(x, w, t, reduction="none", dloss=dloss), dtype)


def test_gradients_of_few_rows_made_with_the_loss():
    """One loss for all rows, few of them: the exponentials are rounded once, what is divided by their sums is not."""
    rows, v, h = 12, 152064, 1024
    x, w, t = inputs(rows, v, h, torch.bfloat16)
    assert made_with_the_loss(x, w, t)
    one = torch.ones((), device="cuda")
    out, want = run(cross_entropy(t, "mean"), x, w, one), plain.losses(x, w, t, dloss=one)
    for name in ("loss", "dx", "dw"):
        plain.within(out[name], want[name], name)
    a, c = x.double(), (t >= 0).double()[:, None] / int((t >= 0).sum())
    q = torch.softmax(a @ w.double().t(), -1).scatter(1, t.clamp(min=0)[:, None], 0.0) * c
    for name, p, m in (("dx", q, w), ("dw", q.t(), a)):
        exact = want[name][0]
        rounded = (exact.bfloat16().double() - exact).norm()
        # Each other word's exponential is off by half a step, 2^-8, and its row's factor by as much; as independent numbers, of which the norm is the root of the sum of squares.
        spread = ((p ** 2) @ (m.double() ** 2)).sum().sqrt()
        assert (out[name].double() - exact).norm() <= 1.1 * rounded + 2.1 * 2.0 ** -8 * spread + 2.0 ** -8 * (p @ m.double()).norm(), name
