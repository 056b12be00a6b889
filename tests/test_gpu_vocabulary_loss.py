"""Losses over a vocabulary whose logits are never stored, and their gradients, against 64 bits."""
import ctypes
import subprocess
import sys
import threading

import pytest
import torch

import nano_nccl_b200 as nn
import plain_vocabulary as plain
from nano_nccl_b200 import ops
from test_cpu_vocabulary_ops import LL, VocabularyLoss
from test_gpu_linear8 import replaced

pytestmark = pytest.mark.gpu
DTYPES = [torch.float32, torch.float16, torch.bfloat16]


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def normal(shape, dtype, seed, scale=1.0):
    return (scale * torch.randn(shape, device="cuda", generator=gen(seed))).to(dtype)


def inputs(rows, vocabulary, width, dtype, seed=0):
    """(x, weight, targets): logits of a standard deviation of two, rows that know their targets and rows that do not, one in seven without."""
    weight = normal((vocabulary, width), dtype, seed, 2.0 / width ** 0.5)
    targets = torch.randint(0, vocabulary, (rows,), device="cuda", generator=gen(seed + 1))
    x = torch.randn(rows, width, device="cuda", generator=gen(seed + 2)) + 3 * torch.rand(rows, 1, device="cuda", generator=gen(seed + 3)) * weight[targets].float()
    targets = torch.where(torch.arange(rows, device="cuda") % 7 == 3, -100, targets)
    return x.to(dtype), weight, targets


def teacher(rows, entries, vocabulary, dtype, seed=0):
    tokens = torch.randint(0, vocabulary, (rows, entries), device="cuda", generator=gen(seed))  # (the same word twice, too)
    return normal((rows, entries), dtype, seed + 1, 3.0) + 5, tokens


def back_of(rows, reduction, seed=9):
    return torch.randn(rows, device="cuda", generator=gen(seed)) if reduction == "none" else torch.tensor(0.75, device="cuda")


def run(call, x, weight, dloss):
    x, weight = x.detach().requires_grad_(), weight.detach().requires_grad_()
    loss = call(x, weight)
    dx, dw = torch.autograd.grad(loss, (x, weight), dloss)
    assert loss.dtype == torch.float32 and dx.dtype == x.dtype and dx.shape == x.shape and dw.shape == weight.shape
    return {"loss": loss.detach(), "dx": dx, "dw": dw}


def check(call, x, weight, targets, reduction, logits=None, temperature=1.0):
    rows = x.shape[:-1].numel()
    dloss = back_of(rows, reduction).reshape(x.shape[:-1] if reduction == "none" else ())
    out = run(call, x, weight, dloss)
    flat = lambda t, n: None if t is None else t.reshape(rows, *t.shape[t.dim() - n:])  # noqa: E731
    want = plain.losses(x.reshape(rows, -1), weight, flat(targets, 0 if logits is None else 1), flat(logits, 1), temperature, reduction, dloss.reshape(-1) if reduction == "none" else dloss)
    for name, value in want.items():
        plain.within(out[name].reshape(value[0].shape), value, name)
    with torch.no_grad():  # (bf16, one loss for all rows: by another way than with gradients)
        loss = call(x, weight)
        plain.within(loss.reshape(want["loss"][0].shape), want["loss"], "loss alone")
        assert torch.equal(loss, out["loss"]) or (x.dtype == torch.bfloat16 and reduction != "none")
    again = run(call, x, weight, dloss)
    assert all(torch.equal(a, b) for a, b in zip(out.values(), again.values()))
    return out


def cross_entropy(targets, reduction):
    return lambda x, w: ops.linear_cross_entropy(x, w, targets, reduction=reduction)


def distillation(logits, tokens, temperature, reduction):
    return lambda x, w: ops.linear_distillation(x, w, logits, tokens, temperature=temperature, reduction=reduction)


# Around a step of 64, half a tile and a tile of 256 on each axis; vocabularies of one word; rows that TMA reads as they lie (width a multiple of 8) and copies.
SHAPES = [(1, 1, 1), (1, 2, 8), (1, 1000, 768), (5, 257, 64), (64, 512, 64), (127, 129, 63), (128, 128, 128), (129, 255, 65), (256, 256, 256), (257, 300, 130), (300, 5000, 72), (1000, 700, 1003),
          (33, 20011, 80), (513, 1025, 392)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,vocabulary,width", SHAPES)
def test_cross_entropy(dtype, rows, vocabulary, width):
    x, w, t = inputs(rows, vocabulary, width, dtype)
    for reduction in ("none", "mean", "sum"):
        check(cross_entropy(t, reduction), x, w, t, reduction)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,vocabulary,width,entries,temperature", [(1, 1, 8, 1, 1.0), (1, 50, 8, 3, 2.0), (33, 257, 64, 1, 1.0), (130, 1009, 80, 7, 1.5), (257, 300, 130, 31, 4.0), (64, 5000, 72, 32, 0.5),
                                                                       (300, 700, 203, 33, 2.0), (20, 600, 264, 256, 3.0)])
def test_distillation(dtype, rows, vocabulary, width, entries, temperature):
    x, w, _ = inputs(rows, vocabulary, width, dtype)
    logits, tokens = teacher(rows, entries, vocabulary, dtype)
    # Entries and whole rows that are not there, by their token and by their logit.
    tokens = torch.where(torch.rand(tokens.shape, device="cuda", generator=gen(3)) < 0.1, -1, tokens)
    logits = torch.where(torch.rand(tokens.shape, device="cuda", generator=gen(4)) < 0.1, -torch.inf, logits)
    tokens[2::11], logits[5::11] = -7, -torch.inf
    for reduction in ("none", "mean"):
        check(distillation(logits, tokens, temperature, reduction), x, w, tokens, reduction, logits, temperature)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,vocabulary,width", [(40, 300, 20000), (2000, 600, 1100), (40000, 300, 72), (70, 60000, 40)])
def test_long_sums(dtype, rows, vocabulary, width):
    """More than 16384 elements of each of the three summed axes (float32: 1024), whole tiles and cut ones."""
    x, w, t = inputs(rows, vocabulary, width, dtype)
    check(cross_entropy(t, "mean"), x, w, t, "mean")


@pytest.mark.parametrize("dtype", DTYPES)
def test_pieces_of_the_vocabulary(dtype):
    """More words than one piece holds: 70000 rows leave 4096 of them to each, 40000 rows (float32: 14000) 6656."""
    for rows, vocabulary in ((70000, 9000), (40000 if dtype != torch.float32 else 14000, 14000)):
        x, w, t = inputs(rows, vocabulary, 72, dtype)
        check(cross_entropy(t, "mean"), x, w, t, "mean")
    logits, tokens = teacher(rows, 5, vocabulary, dtype)
    check(distillation(logits, tokens, 2.0, "mean"), x, w, tokens, "mean", logits, 2.0)


def made_with_the_loss(x, w, t):
    """Whether the gradients of this call are made with the loss: its node has them."""
    calls = []
    prototype = ctypes.CFUNCTYPE(ctypes.c_int, ctypes.c_void_p, ctypes.c_void_p)
    with replaced("b2_vocabulary_loss_both", prototype, lambda original, *arguments: calls.append(1) or original(*arguments)):
        ops.linear_cross_entropy(x.detach().requires_grad_(), w, t)
    return bool(calls)


# bf16, one loss for all rows, a matrix of 2^25 elements at least (256 rows of products are 2^33 then): the logits are made once.
@pytest.mark.parametrize("rows,vocabulary,width", [(1, 50257, 768), (5, 9001, 3800), (257, 33000, 1030), (300, 470000, 72), (1000, 40000, 856), (700, 70001, 1003)])
def test_gradients_made_with_the_loss(rows, vocabulary, width):
    x, w, t = inputs(rows, vocabulary, width, torch.bfloat16)
    assert made_with_the_loss(x, w, t)
    for reduction in ("mean", "sum"):
        check(cross_entropy(t, reduction), x, w, t, reduction)
    logits, tokens = teacher(rows, 33, vocabulary, torch.bfloat16)
    tokens = torch.where(torch.rand(tokens.shape, device="cuda", generator=gen(3)) < 0.1, -1, tokens)
    logits = torch.where(torch.rand(tokens.shape, device="cuda", generator=gen(4)) < 0.1, -torch.inf, logits)
    tokens[2::11], logits[5::11] = -7, -torch.inf
    tokens[:, 3] = tokens[:, 4]  # the same word twice
    check(distillation(logits, tokens, 1.5, "mean"), x, w, tokens, "mean", logits, 1.5)


def test_gradients_made_with_the_loss_by_pieces_of_the_rows():
    """More than 1 GB of exponentials, and a last piece of a few rows more than half."""
    x, w, t = inputs(14001, 40000, 840, torch.bfloat16)
    assert made_with_the_loss(x, w, t)
    check(cross_entropy(t, "mean"), x, w, t, "mean")
    logits, tokens = teacher(14001, 3, 40000, torch.float32)
    check(distillation(logits, tokens, 2.0, "sum"), x, w, tokens, "sum", logits, 2.0)


def test_rows_and_strides_of_gradients_made_with_the_loss():
    b, s, v, h = 2, 60, 40000, 848
    x, w, t = inputs(b * s, v, h + 8, torch.bfloat16)
    x, t = x.view(b, s, h + 8), t.view(b, s)
    check(cross_entropy(t.int(), "mean"), x[..., :h], w[:, :h], t, "mean")
    check(cross_entropy(t, "sum"), x[..., 1:h + 1], w[:, 3:h + 3], t, "sum")
    check(cross_entropy(t[:, ::2], "mean"), x[:, ::2, :h].transpose(0, 1).contiguous().transpose(0, 1), w[:, :h].t().contiguous().t(), t[:, ::2], "mean")
    x, w = x[..., :h].detach(), w[:, :h].detach()
    none = run(cross_entropy(torch.full_like(t, -3), "mean"), x, w, torch.ones((), device="cuda"))
    assert not any(v.any() for v in none.values())
    bad = t.clone()
    bad[1, 7] = v
    out = run(cross_entropy(bad, "mean"), x, w, torch.ones((), device="cuda"))
    assert out["loss"].isnan() and out["dw"].isnan().all() and out["dx"][1, 7].isnan().all() and out["dx"][0].isfinite().all()
    spoilt = x.clone()
    spoilt[0, 3, 5] = float("inf")
    out = run(cross_entropy(t.clamp(min=0), "mean"), spoilt, w, torch.ones((), device="cuda"))
    assert not out["loss"].isfinite() and out["dx"][1].isfinite().all()


@pytest.mark.parametrize("dtype", DTYPES)
def test_strides_and_kinds(dtype):
    b, s, v, h = 3, 50, 300, 96
    x, w, t = inputs(b * s, v, h + 8, dtype)
    x, t = x.view(b, s, h + 8), t.view(b, s)
    check(cross_entropy(t.int(), "none"), x[..., :h], w[:, :h], t, "none")                 # rows further apart
    check(cross_entropy(t, "mean"), x[..., 1:h + 1], w[:, 3:h + 3], t, "mean")             # rows that do not start at 16 bytes
    half = t.clamp(max=149)
    check(cross_entropy(half.t(), "none"), x[..., :h].transpose(0, 1), w[::2, :h], half.t(), "none")
    check(cross_entropy(half[:, ::2], "mean"), x[:, ::2, :h], w[:, :h].t().contiguous().t(), half[:, ::2], "mean")
    check(cross_entropy(t[:, :1].expand(b, s), "mean"), x[:, :1, :h].expand(b, s, h), w[:, :h], t[:, :1].expand(b, s), "mean")
    check(cross_entropy(t[0, 0], "mean"), x[0, 0, :h], w[:, :h], t[0, 0], "mean")
    logits, tokens = teacher(b * s, 12, v, torch.float32)
    logits, tokens = logits.view(b, s, 12), tokens.view(b, s, 12)
    for kind in DTYPES:
        given = logits.to(kind)
        check(distillation(given[..., 1::2], tokens[..., :6].int(), 2.0, "none"), x[..., :h], w[:, :h], tokens[..., :6], "none", given[..., 1::2], 2.0)
    check(distillation(logits[0, 0].expand(b, s, 12), tokens[0, 0].expand(b, s, 12), 1.0, "mean"), x[..., :h], w[:, :h], tokens[0, 0].expand(b, s, 12), "mean", logits[0, 0].expand(b, s, 12))


@pytest.mark.parametrize("dtype", DTYPES)
def test_what_comes_back(dtype):
    """Weights of rows that differ by powers of ten, zeros, strides, and large ones, as a loss scaler has them."""
    rows, v, h = 200, 500, 64
    x, w, t = inputs(rows, v, h, dtype)
    for dloss in (10.0 ** torch.linspace(-4, 0, rows, device="cuda"), torch.zeros(rows, device="cuda"), torch.randn(rows, 2, device="cuda", generator=gen(1))[:, 1], torch.ones(1, device="cuda").expand(rows),
                  torch.randn(rows, device="cuda", generator=gen(2)) * (t % 2)):
        out = run(cross_entropy(t, "none"), x, w, dloss)
        for name, value in plain.losses(x, w, t, reduction="none", dloss=dloss).items():
            plain.within(out[name], value, name)
    for scale in (0.0, -3.0, 1024.0):
        dloss = torch.tensor(scale, device="cuda")
        out = run(cross_entropy(t, "mean"), x, w, dloss)
        for name, value in plain.losses(x, w, t, reduction="mean", dloss=dloss).items():
            plain.within(out[name], value, name)


@pytest.mark.parametrize("dtype", DTYPES)
def test_rows_without_a_target_have_no_gradient(dtype):
    x, w, t = inputs(100, 300, 64, dtype)
    t[40:] = -1
    for reduction in ("none", "mean", "sum"):
        dloss = back_of(100, reduction)
        out = run(cross_entropy(t, reduction), x, w, dloss)
        assert not out["dx"][t < 0].any() and (reduction != "none" or not out["loss"][t < 0].any())
        out = run(cross_entropy(torch.full_like(t, -3), reduction), x, w, dloss)
        assert not out["loss"].any() and not out["dx"].any() and not out["dw"].any()
        # What comes back to them does not matter either.
        if reduction == "none":
            got = run(cross_entropy(t, reduction), x, w, torch.where(t < 0, float("nan"), dloss))
            want = run(cross_entropy(t, reduction), x, w, dloss)
            assert all(torch.equal(got[name], want[name]) for name in got)


def test_words_outside_the_vocabulary_and_infinities():
    x, w, t = inputs(100, 300, 64, torch.bfloat16)
    bad = t.clone()
    bad[17] = 300
    out = run(cross_entropy(bad, "none"), x, w, torch.ones(100, device="cuda"))
    good = run(cross_entropy(t, "none"), x, w, torch.ones(100, device="cuda"))
    others = torch.arange(100, device="cuda") != 17
    assert out["loss"][17].isnan() and out["dx"][17].isnan().all() and out["dw"].isnan().all()
    assert torch.equal(out["loss"][others], good["loss"][others]) and torch.equal(out["dx"][others], good["dx"][others])
    assert ops.linear_cross_entropy(x, w, bad).isnan()
    logits, tokens = teacher(100, 4, 300, torch.bfloat16)
    tokens[17, 2] = 1 << 40
    out = run(distillation(logits, tokens, 1.0, "none"), x, w, torch.ones(100, device="cuda"))
    assert out["loss"][17].isnan() and out["loss"][others].isfinite().all() and out["dx"][17].isnan().all() and out["dx"][others].isfinite().all()
    spoilt = x.clone()
    spoilt[3, 5] = float("inf")
    out = run(cross_entropy(t.clamp(min=0), "none"), spoilt, w, torch.ones(100, device="cuda"))
    others = torch.arange(100, device="cuda") != 3
    assert not out["loss"][3].isfinite() and torch.equal(out["loss"][others & (t >= 0)], good["loss"][others & (t >= 0)]) and out["dx"][others].isfinite().all()


@pytest.mark.parametrize("dtype", DTYPES)
def test_rows_that_are_sure(dtype):
    """Logits far apart: a loss near zero, and one of a few hundred, where sums of exponentials end."""
    rows, v, h = 64, 200, 64
    x, w = torch.zeros(rows, h, device="cuda"), torch.zeros(v, h, device="cuda")
    x[:, 0], w[:, 0] = torch.linspace(0, 30, rows, device="cuda"), torch.linspace(-8, 8, v, device="cuda")
    t = torch.where(torch.arange(rows, device="cuda") % 2 == 0, v - 1, 0)
    out = check(cross_entropy(t, "none"), x.to(dtype), w.to(dtype), t, "none")
    assert (out["loss"] >= 0).all() and out["loss"][-1] > 400 and out["loss"][-2] < 0.2


@pytest.mark.parametrize("c", [4.0, 8.0, 16.0, 40.0])
def test_small_losses_made_with_their_gradients(c):
    """Of rows that are sure of their targets: nothing of what the others leave is lost beside the target's 1."""
    rows, v, h = 200, 530000, 64
    _, w, t = inputs(rows, v, h, torch.bfloat16)
    t[0] = 7
    x = (w[t.clamp(min=0)].float() * c).bfloat16()
    assert made_with_the_loss(x, w, t)
    out = check(cross_entropy(t, "sum"), x, w, t, "sum")
    there = t >= 0
    z = x[there].double() @ w.double().t()
    z = z - z.gather(1, t[there, None])
    others = torch.exp(z).scatter(1, t[there, None], 0.0).sum(-1)
    want = torch.log1p(others).sum()
    # Logits of at most 40 * |w|^2 = 40 * 12: sums of 64 products lose 2^-23 seven times, and their factor of log2(e) rounds once more, of the word's and of the target's. That is what an exponential is off by,
    # relative to itself, and a loss; the rest, additions and roundings in 32 bits, is 64 * 2^-24 of it.
    assert abs(float(out["loss"]) - float(want)) <= (2 * 9 * 2.0 ** -23 * float((x.float().abs() * w[t.clamp(min=0)].float().abs()).sum(-1).max()) * 2 + 64 * 2.0 ** -24) * float(want) + 1e-30


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("c", [4.0, 16.0, 40.0])
def test_small_losses_of_each_row(dtype, c):
    rows, v, h = 70, 2001, 64
    _, w, t = inputs(rows, v, h, dtype)
    x = (w[t.clamp(min=0)].float() * c).to(dtype)
    out = check(cross_entropy(t, "none"), x, w, t, "none")
    there = t >= 0
    z = x[there].double() @ w.double().t()
    z = z - z.gather(1, t[there, None])
    want = torch.log1p(torch.exp(z).scatter(1, t[there, None], 0.0).sum(-1))
    # As above, of each row; float32 sums lose 2^-23 fifteen times and have operands of 22 bits: 24 * 2^-23 at most. Below the normal numbers exponentials are zeros.
    off = 4 * 24 * 2.0 ** -23 * (x[there].float().abs() * w[t[there]].float().abs()).sum(-1).double() + 64 * 2.0 ** -24
    assert ((out["loss"][there].double() - want).abs() <= off * want + v * 2.0 ** -126).all()
    assert (want < 1e-6).any() or c == 4.0


@pytest.mark.parametrize("wide", [False, True])
def test_logits_too_far_above_the_target_s(wide):
    """bf16, one loss for all rows: sums of exponentials over the target's that pass 2^64, in some pieces of the rows and not in others, and a few words over the edge."""
    rows, v, h = (200, 530000, 64) if not wide else (14000, 40000, 840)  # (in two pieces of the rows)
    x, w, t = inputs(rows, v, h, torch.bfloat16)
    assert made_with_the_loss(x, w, t)
    logits, tokens = teacher(rows, 5, v, torch.bfloat16)
    far = x.clone()
    far[rows - 7] = w[5] * 40 * h ** 0.5  # (a logit of word 5 of a few hundred)
    over = t.clone()
    over[rows - 7] = 9
    tokens[tokens == 5] = 6
    calls = [(cross_entropy(over, "mean"), far, over, None, 1.0), (distillation(logits, tokens, 0.5, "sum"), far, tokens, logits, 0.5)]
    if not wide:
        calls += [(cross_entropy(over, "sum"), (far.float() * s).bfloat16(), over, None, 1.0) for s in (0.02, 0.04, 0.05, 0.06, 0.08, 0.5, 2.0)]
    for call, given, targets, kind, tau in calls:
        check(call, given, w, targets, "mean" if call is calls[0][0] else "sum", kind, tau)


@pytest.mark.parametrize("power", [-50, 50])
def test_logits_far_above_the_target_s_of_inputs_that_are_small_or_large(power):
    """Neither the rows over their sums nor the exponentials times the matrix leave the range of the type."""
    rows, v, h = 200, 530000, 64
    x, w, t = inputs(rows, v, h, torch.bfloat16)
    assert made_with_the_loss(x, w, t)
    t[rows - 7] = 9
    for s in (0.02, 0.03, 0.035, 0.045, 0.055):  # (a logit of word 5 of 25 to 70)
        far = x.clone()
        far[rows - 7] = w[5] * 40 * h ** 0.5 * s
        check(cross_entropy(t, "mean"), far * 2.0 ** power, w * 2.0 ** -power, t, "mean")


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("rows", [1, 12])
def test_gradients_of_few_rows_lose_their_own_rounding_alone(dtype, rows):
    x, w, t = inputs(rows, 9000, 4072, dtype)
    logits, tokens = teacher(rows, 12, 9000, dtype)
    for targets, kind, call in ((t, None, cross_entropy(t, "none")), (tokens, logits, distillation(logits, tokens, 1.0, "none"))):
        out = check(call, x, w, targets, "none", kind)
        want = plain.losses(x, w, targets, kind, reduction="none", dloss=back_of(rows, "none"))
        for name in ("dx", "dw"):
            exact = want[name][0]
            rounded = (exact.to(dtype).double() - exact).norm()
            # The softmax is off by what the logits are: sums of 4072 products of about 0.03 that may lose 2^-23 of themselves 64 times, 1e-5 at most beside roundings of at least 2^-13 in the mean,
            # which it makes larger by a tenth at most.
            assert (out[name].double() - exact).norm() <= 1.1 * rounded, name


def test_targets_of_few_rows_made_with_the_loss():
    """The gradient of a target's word loses its own rounding alone, but for what the other rows have of it."""
    rows, v, h = 9, 40065, 2496
    x, w, t = inputs(rows, v, h, torch.bfloat16)
    assert made_with_the_loss(x, w, t)
    out = check(cross_entropy(t, "mean"), x, w, t, "mean")
    one = torch.ones((), device="cuda")
    dw = run(cross_entropy(t, "mean"), x, w, one)["dw"]
    there = t >= 0
    words, a = t[there], x[there].double()
    exact = plain.losses(x, w, t, dloss=one)["dw"][0][words]
    others = torch.softmax(a @ w.double().t(), -1).scatter(1, words[:, None], 0.0)[:, words] / len(words)
    rounded = (exact.bfloat16().double() - exact).norm()
    # (1.1: the softmax, as of few rows above. An element of another row is off by its own rounding and its row's factor, 2^-8 each.)
    assert (dw[words].double() - exact).norm() <= 1.1 * rounded + 2.1 * 2.0 ** -8 * (others.t() @ a.abs()).norm()
    assert out["dw"].shape == w.shape


def test_asking_for_gradients_made_with_the_loss():
    """Twice, apart, multiplied with what comes back, of a loss whose inputs changed."""
    x, w, t = inputs(300, 40000, 856, torch.bfloat16)
    assert made_with_the_loss(x, w, t)
    x, w = x.requires_grad_(), w.requires_grad_()
    loss = ops.linear_cross_entropy(x, w, t)
    one = torch.ones((), device="cuda")
    want = plain.losses(x, w, t, dloss=one)
    (dx,) = torch.autograd.grad(loss, x, retain_graph=True)
    kept = dx.clone()
    (dw,) = torch.autograd.grad(loss, w, retain_graph=True)
    again = torch.autograd.grad(loss, (x, w), retain_graph=True)
    assert torch.equal(dx, kept)
    for name, value in (("dx", dx), ("dw", dw), ("dx", again[0]), ("dw", again[1])):
        plain.within(value, want[name], name)
    for scale in (0.0, 0.5, -3.0, 65536.0, float("nan")):
        got = torch.autograd.grad(ops.linear_cross_entropy(x, w, t) * scale, (x, w))
        for a, b in zip(got, (dx, dw)):
            assert torch.equal(a.nan_to_num(7.0), (b.float() * scale).bfloat16().nan_to_num(7.0))
    loss = ops.linear_cross_entropy(x, w, t)
    with torch.no_grad():
        x.mul_(2.0)
    with pytest.raises(RuntimeError, match="inplace"):
        loss.backward()
    # Two losses of the same matrix in one backward pass.
    first, second = ops.linear_cross_entropy(x, w, t), ops.linear_cross_entropy(x[:100], w, t[:100])
    got = torch.autograd.grad(first + second, w)[0]
    parts = [torch.autograd.grad(ops.linear_cross_entropy(x[:n], w, t[:n]), w)[0] for n in (300, 100)]
    assert torch.equal(got, parts[0] + parts[1])


def test_gradients_by_differences():
    """float32, along a direction: the loss's own rounding is 2^-24 of it, the step 2^-7."""
    x, w, t = inputs(50, 300, 64, torch.float32)
    logits, tokens = teacher(50, 6, 300, torch.float32)
    for call in (cross_entropy(t, "sum"), distillation(logits, tokens, 2.0, "sum")):
        out = run(call, x, w, torch.ones((), device="cuda"))
        step = 2.0 ** -7
        for name, value in (("dx", x), ("dw", w)):
            d = torch.randn(value.shape, device="cuda", generator=gen(8))
            d /= d.norm()
            move = lambda s: call(x + s * d, w) if name == "dx" else call(x, w + s * d)  # noqa: E731
            slope = (move(step).double() - move(-step).double()) / (2 * step)
            want = (out[name].double() * d.double()).sum()
            # Two roundings of the loss over 2 * step, and the third derivative: below the cube of the rows' norms, a step squared.
            bound = 64 * 2.0 ** -24 * out["loss"].double() / step + step ** 2 * (x if name == "dw" else w).double().norm(dim=-1).max() ** 3
            assert (slope - want).abs() <= bound, (name, slope, want, bound)


def test_only_what_is_asked_for():
    x, w, t = inputs(60, 300, 64, torch.bfloat16)
    both = run(cross_entropy(t, "mean"), x, w, torch.ones((), device="cuda"))
    xg, wg = x.clone().requires_grad_(), w.clone().requires_grad_()
    (dx,) = torch.autograd.grad(ops.linear_cross_entropy(xg, w, t), xg)
    (dw,) = torch.autograd.grad(ops.linear_cross_entropy(x, wg, t), wg)
    (first,) = torch.autograd.grad(ops.linear_cross_entropy(xg, wg, t), xg)
    assert torch.equal(dx, both["dx"]) and torch.equal(dw, both["dw"]) and torch.equal(first, dx)
    loss = ops.linear_cross_entropy(xg, wg, t)
    with torch.no_grad():
        wg.mul_(2.0)
    with pytest.raises(RuntimeError, match="inplace"):
        loss.backward()
    (dx,) = torch.autograd.grad(ops.linear_cross_entropy(xg, wg, t), xg, create_graph=True)
    with pytest.raises(RuntimeError, match="second derivative"):
        dx.sum().backward()
    # No rows at all.
    empty = x[:0].clone().requires_grad_()
    for reduction, shape in (("none", (0,)), ("mean", ()), ("sum", ())):
        loss = ops.linear_cross_entropy(empty, wg, t[:0], reduction=reduction)
        dx, dw = torch.autograd.grad(loss, (empty, wg), torch.ones_like(loss))
        assert loss.shape == shape and not loss.any() and dx.shape == (0, 64) and dw.shape == wg.shape and not dw.any()


def test_refusals():
    x, w, t = inputs(6, 30, 64, torch.bfloat16)
    logits, tokens = teacher(6, 4, 30, torch.float32)
    for call in (lambda: ops.linear_cross_entropy(x, w, t[:5]), lambda: ops.linear_cross_entropy(x, w, t[:, None]), lambda: ops.linear_cross_entropy(x, w[:, :63], t), lambda: ops.linear_cross_entropy(x, w.half(), t),
                 lambda: ops.linear_cross_entropy(x.double(), w.double(), t), lambda: ops.linear_cross_entropy(x, w, t.float()), lambda: ops.linear_cross_entropy(x, w[:0], t), lambda: ops.linear_cross_entropy(x, w[0], t),
                 lambda: ops.linear_cross_entropy(x[:, :0], w[:, :0], t), lambda: ops.linear_cross_entropy(x, w.cpu(), t), lambda: ops.linear_distillation(x, w, logits, tokens[:, :3]),
                 lambda: ops.linear_distillation(x, w, logits[:, :0], tokens[:, :0]), lambda: ops.linear_distillation(x, w, logits[:, :1].expand(6, 257), tokens[:, :1].expand(6, 257)),
                 lambda: ops.linear_distillation(x, w, logits.double(), tokens), lambda: ops.linear_distillation(x, w, tokens, tokens), lambda: ops.linear_distillation(x, w, logits.requires_grad_(), tokens)):
        with pytest.raises(ValueError):
            call()


@pytest.mark.parametrize("kind", [torch.float16, torch.bfloat16])
def test_autocast_casts_as_linear(kind):
    x, w, t = inputs(60, 300, 64, torch.float32)
    x, w = x.requires_grad_(), w.requires_grad_()
    with torch.autocast("cuda", dtype=kind):
        loss = ops.linear_cross_entropy(x, w, t)
    dx, dw = torch.autograd.grad(loss, (x, w))
    want = run(cross_entropy(t, "mean"), x.to(kind), w.to(kind), torch.ones((), device="cuda"))
    assert torch.equal(loss, want["loss"]) and torch.equal(dx, want["dx"].float()) and torch.equal(dw, want["dw"].float())


def test_captured_calls_and_other_streams():
    """Two graphs of losses with their gradients, replayed at once with eager calls on a third stream, on inputs of their own that change."""
    rows, v, h = 300, 2000, 136
    streams = [torch.cuda.Stream() for _ in range(3)]
    states, graphs, outs = [], [], []
    for i, s in enumerate(streams):
        x, w, t = inputs(rows, v, h, torch.bfloat16, seed=10 * i)
        logits, tokens = teacher(rows, 9, v, torch.bfloat16, seed=10 * i)
        call = cross_entropy(t, "mean") if i != 1 else distillation(logits, tokens, 2.0, "none")
        states.append((call, x, w, back_of(rows, "mean" if i != 1 else "none"), t))
    torch.cuda.synchronize()
    for s, state in zip(streams[:2], states):
        with torch.cuda.stream(s):
            run(*state[:4])
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            outs.append(run(*state[:4]))
        graphs.append(graph)
    for turn in range(3):
        for i, state in enumerate(states):
            state[1].copy_(inputs(rows, v, h, torch.bfloat16, seed=100 * turn + i)[0])
        want = [run(*state[:4]) for state in states]
        torch.cuda.synchronize()
        for s, graph in zip(streams, graphs):
            with torch.cuda.stream(s):
                graph.replay()
        with torch.cuda.stream(streams[2]):
            third = run(*states[2][:4])
        torch.cuda.synchronize()
        for got, expected in zip((*outs, third), want):
            assert all(torch.equal(got[name], expected[name]) for name in expected)


def test_a_matrix_past_32_bits():
    """More than 2^31 elements of the matrix and 2^32 bytes of its gradient; words at its ends."""
    v, h, rows = (1 << 19) + 77, 4104, 20
    assert v * h > 1 << 31
    w = torch.zeros(v, h, dtype=torch.bfloat16, device="cuda")
    w[-300:] = normal((300, h), torch.bfloat16, 1, 2.0 / h ** 0.5)
    x = normal((rows, h), torch.bfloat16, 2)
    t = v - 1 - torch.arange(rows, device="cuda") * 13
    out = run(cross_entropy(t, "sum"), x, w, torch.ones((), device="cuda"))
    # All words but the last 300 have logits of zero: one sum, and the same gradient.
    z = x.double() @ w[-300:].double().t()
    top = z.max(-1, keepdim=True).values.clamp(min=0)
    total = torch.exp(z - top).sum(-1, keepdim=True) + (v - 300) * torch.exp(-top)
    loss = (top + total.log() - z.gather(1, (t - (v - 300))[:, None])).sum()
    assert abs(out["loss"].double() - loss) <= 2.0 ** -18 * loss
    p = torch.exp(z - top) / total
    p.scatter_add_(1, (t - (v - 300))[:, None], -torch.ones(rows, 1, dtype=torch.float64, device="cuda"))
    size = p.abs().t() @ x.double().abs()
    assert ((out["dw"][-300:].double() - p.t() @ x.double()).abs() <= 2.0 ** -6 * size + 1e-30).all()
    flat = (torch.exp(-top) / total).t() @ x.double()
    size = (torch.exp(-top) / total).t() @ x.double().abs()
    assert ((out["dw"][0].double() - flat).abs() <= 2.0 ** -6 * size).all() and (out["dw"][:-300] == out["dw"][0]).all()
    assert ((out["dx"].double() - p @ w[-300:].double()).abs() <= 2.0 ** -6 * (p.abs() @ w[-300:].double().abs())).all()


def called(x, w, t, dloss, wait_ns, kept=None):
    """The C interface: the loss's gradient with waits of `wait_ns`, or the loss itself (kept None): (loss or (dx, dw), kept)."""
    lib, rows = nn.load(), x.shape[0]
    loss, dx, dw = torch.zeros(rows, device="cuda"), torch.zeros_like(x), torch.zeros_like(w)
    c = VocabularyLoss(dtype=2, x=x.data_ptr(), x_stride=x.stride(0), weight=w.data_ptr(), weight_stride=w.stride(0), tokens=rows, width=x.shape[1], vocabulary=w.shape[0], targets=t.data_ptr(),
                       target_bytes=8, target_strides=(LL * 2)(1, 1), temperature=1.0, loss=loss.data_ptr(), loss_grad=dloss.data_ptr(), loss_grad_stride=1, x_grad=dx.data_ptr(),
                       weight_grad=dw.data_ptr())
    backward = kept is not None
    floats, size = ctypes.c_size_t(), ctypes.c_size_t()
    assert lib.b2_vocabulary_loss_sizes(ctypes.byref(c), int(backward), ctypes.byref(floats), ctypes.byref(size)) == 0
    kept = torch.empty(floats.value, device="cuda") if kept is None else kept
    workspace = torch.empty(size.value, dtype=torch.uint8, device="cuda")
    c.kept, c.workspace = kept.data_ptr(), workspace.data_ptr()
    stream = ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)
    assert lib.b2_vocabulary_loss_within(ctypes.byref(c), int(backward), ctypes.c_ulonglong(wait_ns), stream) == 0
    torch.cuda.synchronize()
    return ((dx, dw) if backward else loss), kept


def test_a_wait_that_runs_out_leaves_nan():
    """Without any time a wait makes two polls all the same, of a microsecond or more, and may be over by then (it is for a few microseconds): a call's results are the right ones or NaN, its status
    says which, and of many calls some run out."""
    x, w, t = inputs(4096, 1024, 32768, torch.bfloat16)
    t, dloss = t.clamp(min=0), torch.ones(4096, device="cuda")
    ops.check_async_error()
    want, kept = called(x, w, t, dloss, 2 * 10 ** 9)
    grads, _ = called(x, w, t, dloss, 2 * 10 ** 9, kept)
    assert want.isfinite().all() and all(g.isfinite().all() for g in grads)

    def ran_out():
        try:
            ops.check_async_error()
        except nn.B200CclError as e:
            assert "ran out" in str(e)
            ops.check_async_error()  # (it is said once)
            return True
        return False

    seen = [0, 0]
    for _ in range(60):
        loss, _ = called(x, w, t, dloss, 0)
        nan = loss.isnan()
        assert torch.equal(loss[~nan], want[~nan]) and bool(nan.any()) == ran_out()
        seen[0] += bool(nan.any())
        got, _ = called(x, w, t, dloss, 0, kept)
        if ran_out():
            assert all(g.isnan().all() for g in got)
            seen[1] += 1
        else:
            assert all(torch.equal(a, b) for a, b in zip(got, grads))
    assert min(seen) > 0
    # Nobody else is told.
    assert torch.equal(called(x, w, t, dloss, 2 * 10 ** 9)[0], want)
    assert all(torch.equal(a, b) for a, b in zip(called(x, w, t, dloss, 2 * 10 ** 9, kept)[0], grads))
    assert not ran_out()


def test_a_failure_in_a_backward_pass_is_this_library_s_error():
    x, w, t = inputs(6, 30, 64, torch.float32)
    prototype = ctypes.CFUNCTYPE(ctypes.c_int, ctypes.c_void_p, ctypes.c_void_p)
    with replaced("b2_vocabulary_loss_backward", prototype, lambda original, *arguments: 1):
        with pytest.raises(nn.B200CclError):
            ops.linear_cross_entropy(x.requires_grad_(), w, t).backward()
    with replaced("b2_vocabulary_loss_forward", prototype, lambda original, *arguments: 1):
        with pytest.raises(nn.B200CclError):
            ops.linear_cross_entropy(x, w, t)
    x, w, t = inputs(6, 40000, 856, torch.bfloat16)
    with replaced("b2_vocabulary_loss_times", prototype, lambda original, *arguments: 1):
        with pytest.raises(nn.B200CclError):
            ops.linear_cross_entropy(x.requires_grad_(), w, t).backward()


def test_only_one_gradient_made_with_the_loss():
    x, w, t = inputs(300, 40000, 856, torch.bfloat16)
    assert made_with_the_loss(x, w, t)
    one = torch.ones((), device="cuda")
    both = run(cross_entropy(t, "mean"), x, w, one)
    xg, wg = x.clone().requires_grad_(), w.clone().requires_grad_()
    (dx,) = torch.autograd.grad(ops.linear_cross_entropy(xg, w, t), xg)
    (dw,) = torch.autograd.grad(ops.linear_cross_entropy(x, wg, t), wg)
    assert torch.equal(dx, both["dx"]) and torch.equal(dw, both["dw"])
    # A gradient that nobody asks for is left where it is.
    loss = ops.linear_cross_entropy(xg, wg, t)
    (dx,) = torch.autograd.grad(loss * 2, xg)
    assert torch.equal(dx, both["dx"] * 2)


def test_graphs_of_gradients_made_with_the_loss():
    """Two graphs at once, with what comes back in memory that changes; and a backward pass in a graph whose loss was made before it."""
    graphs, states, streams = [], [], [torch.cuda.Stream() for _ in range(2)]
    for i, s in enumerate(streams):
        x, w, t = inputs(200, 40000, 856, torch.bfloat16, seed=10 * i)
        back = torch.tensor(1.0, device="cuda")
        logits, tokens = teacher(200, 9, 40000, torch.bfloat16, seed=i)
        call = cross_entropy(t, "mean") if i == 0 else distillation(logits, tokens, 2.0, "sum")
        torch.cuda.synchronize()
        with torch.cuda.stream(s):
            run(call, x, w, back)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            out = run(call, x, w, back)
        graphs.append(graph)
        states.append((call, x, w, back, out))
    for turn in range(4):
        for i, (call, x, w, back, out) in enumerate(states):
            x.copy_(inputs(200, 40000, 856, torch.bfloat16, seed=100 * turn + i)[0])
            back.fill_((1.0, 0.3, 1.0, -2.0)[turn])
        want = [run(*state[:4]) for state in states]
        torch.cuda.synchronize()
        for s, graph in zip(streams, graphs):
            with torch.cuda.stream(s):
                graph.replay()
        torch.cuda.synchronize()
        for state, expected in zip(states, want):
            assert all(torch.equal(state[4][name], expected[name]) for name in expected)
    call, x, w, back, _ = states[0]
    x, w = x.clone().requires_grad_(), w.clone().requires_grad_()
    s = streams[0]
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        loss = call(x, w)
    torch.cuda.synchronize()
    back.fill_(0.5)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        grads = torch.autograd.grad(loss, (x, w), back, retain_graph=True)
    want = plain.losses(x, w, inputs(200, 40000, 856, torch.bfloat16, seed=0)[2], dloss=torch.tensor(0.5, device="cuda"))
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        for name, g in zip(("dx", "dw"), grads):
            plain.within(g, want[name], name)


def test_a_graph_of_the_loss_and_one_of_its_backward_pass():
    """The second may be replayed more often than the first."""
    x, w, t = inputs(200, 40000, 856, torch.bfloat16)
    s = torch.cuda.Stream()
    back = torch.tensor(0.3, device="cuda")
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        expected = run(cross_entropy(t, "mean"), x, w, back)
    torch.cuda.synchronize()
    want = plain.losses(x, w, t, dloss=back)
    x.requires_grad_()
    w.requires_grad_()
    first, second = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(first, stream=s):
        loss = ops.linear_cross_entropy(x, w, t)
    with torch.cuda.graph(second, stream=s, pool=first.pool()):
        grads = torch.autograd.grad(loss, (x, w), back)
    for _ in range(2):
        first.replay()
        for _ in range(2):
            second.replay()
            torch.cuda.synchronize()
            assert torch.equal(loss, expected["loss"])
            for name, g in zip(("dx", "dw"), grads):
                plain.within(g, want[name], name)


FIRST_INSIDE_A_CAPTURE = """
import torch
from nano_nccl_b200 import ops
torch.cuda.init()
w = torch.randn(300, 64, device="cuda").bfloat16().requires_grad_()
t = torch.randint(0, 300, (50,), device="cuda")
s = torch.cuda.Stream()
s.wait_stream(torch.cuda.current_stream())
with torch.cuda.stream(s):  # (torch's own first calls)
    torch.autograd.grad((w * 2).float().sum(), w)
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
def step():
    loss = ops.linear_cross_entropy(ops.embedding(t, w, 8.0), w, t)
    return loss, torch.autograd.grad(loss, w)[0]
with torch.cuda.graph(graph, stream=s):
    captured = step()
graph.replay()
torch.cuda.synchronize()
want = step()
assert torch.equal(captured[0], want[0]) and torch.equal(captured[1], want[1])
print("the same")
"""


def test_first_calls_inside_a_capture():
    done = subprocess.run([sys.executable, "-c", FIRST_INSIDE_A_CAPTURE], capture_output=True, text=True, timeout=240)
    assert done.returncode == 0 and "the same" in done.stdout, done.stderr


def test_calls_of_several_threads():
    """Each on a stream of its own, at the same time, with gradients."""
    results, wanted = [None] * 4, []
    states = []
    for i in range(4):
        x, w, t = inputs(150 + i, 3000, 136, (torch.bfloat16, torch.float32)[i % 2], seed=i)
        states.append((cross_entropy(t, "mean"), x, w, torch.ones((), device="cuda")))
        wanted.append(run(*states[-1]))
    torch.cuda.synchronize()

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(10):
                out = run(*states[i])
            torch.cuda.current_stream().synchronize()
        results[i] = out

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for thread in threads:
        thread.start()
    for thread in threads:
        thread.join()
    for got, want in zip(results, wanted):
        assert got is not None and all(torch.equal(got[name], want[name]) for name in want)


def test_transformations_are_refused():
    x, w, t = inputs(4, 30, 64, torch.float32)
    with pytest.raises((RuntimeError, ValueError)):
        torch.func.vmap(lambda a: ops.linear_cross_entropy(a, w, t))(x.expand(2, 4, 64))
    with pytest.raises((RuntimeError, ValueError)):
        torch.func.vmap(lambda a: ops.embedding(t, a))(w.expand(2, 30, 64))
    with pytest.raises((RuntimeError, ValueError)):
        torch.func.grad(lambda a: ops.linear_cross_entropy(a, w, t))(x)
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(x, torch.ones_like(x))
        with pytest.raises(ValueError, match="tangent"):
            ops.linear_cross_entropy(dual, w, t)
        with pytest.raises(ValueError, match="tangent"):
            ops.embedding(t, dual)
