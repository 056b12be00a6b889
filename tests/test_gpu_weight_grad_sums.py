"""Weight gradients of long sums: what the additions leave of them, against sums in 64 bits."""
import pytest
import torch

import plain8
from nano_nccl_b200 import ops

pytestmark = pytest.mark.gpu


def product(dy, x):
    """dy^T x in 64 bits."""
    want = torch.zeros(dy.shape[1], x.shape[1], dtype=torch.float64, device="cuda")
    for i in range(0, dy.shape[0], 1 << 16):
        want += dy[i:i + (1 << 16)].double().t() @ x[i:i + (1 << 16)].double()
    return want


def one_sign(tokens, inputs, outputs, dtype):
    """Positive dY, each output under a scale of its own, and positive inputs that 8 bits hold exactly."""
    gen = torch.Generator(device="cuda").manual_seed(tokens)
    x = torch.randint(1, 128, (tokens, inputs), device="cuda", generator=gen).to(dtype) / 64
    x[:, ::32] = 127 / 64
    scale = 2.0 ** (torch.rand(outputs, device="cuda", generator=gen) - 14.0)
    dy = ((torch.rand(tokens, outputs, device="cuda", generator=gen) + 0.5) * scale).to(dtype)
    return dy, x


# Tiles of 256 outputs, cut and whole; of 512 outputs, cut, and whole ones in two waves. Lengths that end inside a step.
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("tokens,inputs,outputs", [(2000003, 64, 64), (300011, 256, 4096), (262144, 2048, 2560), (70001, 4096, 4096), (262144, 4096, 2560)])
def test_long_sums_of_one_sign(dtype, tokens, inputs, outputs):
    dy, x = one_sign(tokens, inputs, outputs, dtype)
    p = ops.pack8(x)
    assert torch.equal(ops.unpack8(p), x)
    dw, _ = ops.weight_grad8(dy, p)
    want = product(dy, x)
    error = (dw.double() - want) / want
    # The tensor cores add 16 products to the sum so far in one instruction: each product is cut at a quarter of the last of 24 bits of the sum, their
    # total at the whole: 5 units of 2^-23 at most. Over the 1024 instructions of 16384 tokens, whose sums grow evenly, 5 * 512 * 2^-23 of the result; half of
    # it on average. Adding such sums to one another rounds: 250 times 2^-24. Then one rounding to the type.
    sums = 5 * 512 * 2.0 ** -23 + 250 * 2.0 ** -24
    half = plain8.half_step(dtype)
    assert (error.abs() <= half + sums).all()
    # What all results have in common: no more than that half, and what is left of the mean of so many roundings.
    assert error.mean().abs() <= sums / 2 + 5 * half / 3 ** 0.5 / outputs ** 0.5


# Few features, so that one tile sums every step, and many; one tile, cut, and as many as stay whole; parts of a chunk and of a step at the end.
@pytest.mark.parametrize("sign", ["one", "both"])
@pytest.mark.parametrize("tokens,inputs,outputs", [(1025, 32, 8), (8192, 768, 2304), (26001, 700, 500), (200003, 64, 64), (70000, 32, 9000), (500009, 300, 130)])
def test_bias_of_full_precision(tokens, inputs, outputs, sign):
    gen = torch.Generator(device="cuda").manual_seed(tokens)
    dy = torch.rand(tokens, outputs, device="cuda", generator=gen) + 0.5
    if sign == "both":
        dy *= torch.randint(0, 2, dy.shape, device="cuda", generator=gen) * 2 - 1
    x = torch.ones(tokens, inputs, device="cuda")
    _, db = ops.weight_grad8(dy, ops.pack8(x), bias=True)
    want, most = (sum(t[i:i + (1 << 16)].double().sum(0) for i in range(0, tokens, 1 << 16)) for t in (dy, dy.abs()))
    # Steps of 64 tokens: 20 roundings, of each of dY's three parts; what comes behind them is added exactly. Then shares of at most 36 tiles and
    # pairs, eight of them in one row, and a rounding.
    assert ((db.double() - want).abs() <= (20 + 20) * 2.0 ** -24 * most).all()


# Tiles of 256 and 512 outputs, whole and cut, side by side and not, one and several waves, few and many tokens.
PLANS = [(26001, 700, 500), (20000, 1100, 260), (9000, 513, 4700), (16000, 64, 64), (12007, 29, 2227), (15126, 320, 61), (20000, 4096, 5000), (8192, 2048, 2048),
         (1025, 4096, 4700), (40961, 512, 1536)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("tokens,inputs,outputs", PLANS)
def test_every_plan_is_exact_where_sums_are(dtype, tokens, inputs, outputs):
    """Whole numbers whose sums stay below 2^24: a step of tokens lost, taken twice or added to another tile shows, and so does a share of the bias."""
    gen = torch.Generator(device="cuda").manual_seed(tokens)
    x = torch.randint(-3, 4, (tokens, inputs), device="cuda", generator=gen).to(dtype)
    x[:, ::32] = 64
    dy = torch.randint(-2, 3, (tokens, outputs), device="cuda", generator=gen).to(dtype)
    assert 64 * 2 * tokens < 1 << 24
    dw, db = ops.weight_grad8(dy, ops.pack8(x), bias=True)
    assert torch.equal(dw, product(dy, x).to(dtype)) and torch.equal(db, dy.double().sum(0).to(dtype))
    again, none = ops.weight_grad8(dy, ops.pack8(x))
    assert torch.equal(again, dw) and none is None


@pytest.mark.parametrize("tokens,inputs,outputs", [(1, 40, 30), (1025, 300, 700), (2048, 64, 64), (8192, 768, 2304), (15126, 320, 611), (1025, 4096, 4700), (8200, 1100, 5000), (100003, 96, 2000)])
def test_every_part_of_float32_reaches_its_token(tokens, inputs, outputs):
    """One number of 24 bits, of its own size, for each output, at a token that no other has (as far as there are so many): every result is exact, and
    any of the three parts that met another token's inputs would show."""
    gen = torch.Generator(device="cuda").manual_seed(outputs)
    token = (torch.arange(outputs, device="cuda") * max(1, tokens // outputs) + torch.randint(0, max(1, tokens // outputs), (outputs,), device="cuda", generator=gen)) % tokens
    token[-1] = tokens - 1
    number = (torch.randint(1 << 22, 1 << 23, (outputs,), device="cuda", generator=gen) * 2 + 1).float()
    number *= 2.0 ** torch.randint(-40, 20, (outputs,), device="cuda", generator=gen) * (torch.randint(0, 2, (outputs,), device="cuda", generator=gen) * 2 - 1)
    dy = torch.zeros(tokens, outputs, device="cuda")
    dy[token, torch.arange(outputs, device="cuda")] = number
    # Powers of two that tell tokens apart, and blocks of features.
    power = torch.arange(tokens, device="cuda")[:, None] * 7 % 11 + torch.arange(inputs, device="cuda")[None, :] // 32 % 5
    x = 2.0 ** power.float()
    dw, db = ops.weight_grad8(dy, ops.pack8(x), bias=True)
    assert torch.equal(dw, number[:, None] * x[token]) and torch.equal(db, number)


@pytest.mark.parametrize("tokens,inputs,outputs", [(8192, 768, 2304), (26001, 700, 500), (20000, 1100, 260), (16000, 64, 64), (2048, 64, 64), (65536, 512, 512)])
def test_full_precision_of_long_sums(tokens, inputs, outputs):
    gen = torch.Generator(device="cuda").manual_seed(inputs)
    dy, x = torch.randn(tokens, outputs, device="cuda", generator=gen), torch.randn(tokens, inputs, device="cuda", generator=gen)
    p = ops.pack8(x)
    dw, db = ops.weight_grad8(dy, p, bias=True)
    # T additions of both signs in a row, rounded to 24 bits, are off by 2^-24 / sqrt(3) * sqrt(T / 2) of the norm: 1.1e-6 for 2048 terms, more for more.
    # The kernel adds in chunks and may not be worse than that. (dY cut to 8 bits would be off by 2^-8, to 16 by 2^-16.)
    for got, want in ((dw, product(dy, ops.unpack8(p))), (db, dy.double().sum(0))):
        assert (got.double() - want).norm() <= 1e-6 * want.norm()
