"""Plain 64-bit forms of the training operators, for their tests."""
import math

import torch


def kept(x, block=32):
    """What the 8-bit form of `x` stands for, in 64 bits on the CPU: blocks of `block` elements of the last axis."""
    low = -24 if x.dtype == torch.float16 else -126
    v = x.detach().double().cpu()
    columns = v.shape[-1]
    rows = torch.nn.functional.pad(v.reshape(-1, columns), (0, -columns % block)).reshape(-1, block)
    out = torch.empty_like(rows)
    for i, row in enumerate(rows):
        amax = row.abs().max().item()
        if not math.isfinite(amax):
            out[i] = math.nan
            continue
        q = max(math.frexp(amax)[1] - 7, low) if amax > 0 else low
        out[i] = torch.sign(row) * torch.round(row.abs() * 2.0 ** -q).clamp(max=127.0) * 2.0 ** q
    return out.reshape(-1, columns + -columns % block)[:, :columns].reshape(v.shape)


def half_step(dtype):
    """Relative error of one rounding."""
    return torch.finfo(dtype).eps / 2


def gelu(x, tanh):
    if tanh:
        # (1 + tanh u) / 2, without the difference that even 64 bits lose far out
        return x * torch.sigmoid(2.0 * math.sqrt(2.0 / math.pi) * (x + 0.044715 * x ** 3))
    return 0.5 * x * torch.special.erfc(-x / math.sqrt(2.0))


def rotate(x, positions, frequencies, interleaved, magnitude):
    """x [batch, tokens, heads, dim] and positions [tokens] or [batch, tokens], all in 64 bits."""
    n = frequencies.numel()
    angle = positions.double().reshape(-1 if positions.dim() == 2 else 1, x.shape[1], 1, 1) * frequencies.double()
    if positions.dim() == 1:
        angle = angle.expand(x.shape[0], -1, -1, -1)
    c, s = magnitude * angle.cos(), magnitude * angle.sin()
    out = x.clone()
    for i in range(n):
        a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + n)
        u, v = x[..., a], x[..., b]
        out[..., a] = u * c[..., i] - v * s[..., i]
        out[..., b] = u * s[..., i] + v * c[..., i]
    return out
