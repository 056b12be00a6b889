"""Plain 64-bit forms of the operators over a vocabulary, with bounds of what their kernels may be off by, for their tests."""
import torch


def half_step(dtype):
    """Relative error of one rounding."""
    return torch.finfo(dtype).eps / 2


def smallest(dtype):
    """Absolute error of a rounding below the normal numbers."""
    return torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2


def embedding_gradient(tokens, dy, vocabulary, scale):
    """(dw, bound): sums in 32 bits, rounded once."""
    width = dy.shape[-1]
    tokens, rows = tokens.reshape(-1).long(), dy.detach().reshape(-1, width).double()
    there = (tokens >= 0) & (tokens < vocabulary)
    tokens, rows = tokens[there], rows[there]
    dw, size = (torch.zeros(vocabulary, width, dtype=torch.float64, device=dy.device) for _ in range(2))
    dw.index_add_(0, tokens, rows)
    size.index_add_(0, tokens, rows.abs())
    # Each addition rounds a partial sum, which is at most the sum of the magnitudes; then the product with the scale and one rounding.
    additions = torch.bincount(tokens, minlength=vocabulary).double()[:, None]
    dw, size = dw * scale, size * abs(scale)
    return dw, (additions + 2) * 2.0 ** -24 * size + half_step(dy.dtype) * dw.abs() + smallest(dy.dtype)


def _sums(dtype, summed):
    """Relative error (of the sum of the magnitudes) of a product's sum on the tensor cores: an instruction adds 16 products and may cut a step of 24 bits of the sum so far, at most 1024 of
    them in 16-bit types and 3 * 64 in float32 before sums are added up in memory, rounded. float32: both operands are two fp16 numbers, within 2^-22, and the product of the
    second ones, 2^-22, is left out."""
    if dtype == torch.float32:
        return (3 * (min(summed, 1024) / 16 + 1) + summed / 1024 + 4) * 2.0 ** -23 + 3 * 2.0 ** -22
    return (min(summed, 16384) / 16 + summed / 16384 + 3) * 2.0 ** -23


def _floor(dtype, t):
    """What the second fp16 number of a float32 one may be off by at least: half of 2^-24, scaled by a power of two that brings the largest element to 2^14 at least."""
    return 2.0 ** -39 * t.abs().max() if dtype == torch.float32 else 0.0


def losses(x, weight, targets, teacher_logits=None, temperature=1.0, reduction="mean", dloss=None):
    """{"loss", "dx", "dw"}: pairs of a value in 64 bits and the bound of its error. x: [rows, width], all on one device."""
    dtype, (rows, width), vocabulary = x.dtype, x.shape, weight.shape[0]
    a, w, h = x.detach().double(), weight.detach().double(), half_step(x.dtype)
    z = a @ w.t() / temperature
    off = _sums(dtype, width) * (a.abs() @ w.abs().t()) / temperature  # of each logit
    off = off + (_floor(dtype, a) * w.abs().sum(-1)[None] + _floor(dtype, w) * a.abs().sum(-1)[:, None]) / temperature
    off = off.max(-1, keepdim=True).values
    lse = torch.logsumexp(z, -1, keepdim=True)
    q = torch.exp(z - lse)
    if teacher_logits is None:
        entries, there = targets[:, None].clamp(min=0).long(), targets[:, None] >= 0
        y, log_y = there.double(), torch.zeros_like(entries, dtype=torch.float64)
    else:
        entries, there = targets.clamp(min=0).long(), (targets >= 0) & (teacher_logits > -torch.inf)
        t = (teacher_logits.double() / temperature).masked_fill(~there, -torch.inf)
        log_y = torch.log_softmax(t, -1).masked_fill(~there, 0.0)
        y = torch.where(there, log_y.exp(), 0.0)
    counted = there.any(-1)
    each = temperature ** 2 * (y * (log_y - z.gather(1, entries) + lse)).sum(-1)
    each = torch.where(counted, each, 0.0)
    # The logits' own errors, twice; differences, logarithms and the teacher's softmax in 32 bits; the sum over the vocabulary (exponentials within 2 steps, additions of 32, then tiles).
    magnitude = z.abs().max(-1).values + lse.squeeze(-1).abs() + log_y.abs().max(-1).values + 1.0
    if teacher_logits is not None:
        magnitude = magnitude + teacher_logits.double().masked_fill(~there, 0.0).abs().max(-1).values / temperature
    relative = 2 * off.squeeze(-1) + 64 * 2.0 ** -24 * magnitude
    each_off = temperature ** 2 * relative * counted * (1 if teacher_logits is None else 2)
    count = max(1, int(counted.sum())) if reduction == "mean" else 1
    out = {"loss": (each, each_off)}
    if reduction != "none":
        total = each.sum() / count
        out["loss"] = (total, each_off.sum() / count + (rows / 1024 + 16) * 2.0 ** -24 * each.abs().sum() / count)
    if dloss is None:
        return out
    c = temperature * counted[:, None] * (dloss.double() / count if reduction != "none" else dloss.double()[:, None])
    dz = q.scatter_add(1, entries, -y) * c
    # Of an element of P: its own rounding (float32: two fp16 numbers), and what the softmax is off by; in fp16 it is held as 2^14 times its share of the largest row's.
    element = dz.abs() * (h if dtype != torch.float32 else 2.0 ** -22) + c.abs() * q * relative[:, None]
    element = element.scatter_add(1, entries, y * c.abs() * (0.0 if teacher_logits is None else 1.0) * relative[:, None])
    if dtype != torch.bfloat16:
        element = element + c.abs().max() * 2.0 ** -14 * smallest(torch.float16)
    element = element + 2.0 ** -126
    # bf16, one loss for all rows: a row has a factor that makes its target's element, or those of its entries, the ones that are rounded least. It is v / bf16(v) for some v, within h of 1, and the
    # other elements, rounded on their own (h, above), are multiplied by it: (1 + h) (1 + h) - 1 is h and h (1 + h).
    made_with_the_loss = dtype == torch.bfloat16 and reduction != "none"
    if made_with_the_loss:
        element = element + h * (1 + h) * dz.abs()
    for name, p, e, m, summed in (("dx", dz, element, w, vocabulary), ("dw", dz.t(), element.t(), a, rows)):
        exact = p @ m
        sums = p.abs() @ m.abs()
        # bf16, one loss for all rows: what is multiplied with x is 1 / S of P's row, S times P beside x / S, which is rounded as P is. Once in the sum of magnitudes, then.
        # And what comes back to the loss is multiplied with a rounded gradient, and the product rounded.
        sums_of_rounded = h * (sums + e @ m.abs()) if name == "dw" and made_with_the_loss else 0.0
        roundings = (2 + h) if made_with_the_loss else 1
        out[name] = (exact, sums_of_rounded + e @ m.abs() + _floor(dtype, m) * p.abs().sum(-1, keepdim=True) + (_sums(dtype, summed) + 16 * 2.0 ** -24) * sums + roundings * h * (exact.abs() + sums_of_rounded + e @ m.abs()) + smallest(dtype))
    return out


def within(got, wanted, what=""):
    value, bound = wanted
    off = (got.double() - value).abs()
    assert torch.isfinite(got).all(), what
    worst = (off / bound).max() if off.numel() else torch.zeros(())
    assert (off <= bound).all(), f"{what}: {float(worst):.3g} times its bound"
