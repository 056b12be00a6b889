"""Lookup in an embedding and its gradient, against 64 bits."""
import pytest
import torch

import nano_nccl_b200 as nn
import plain_vocabulary as plain
from nano_nccl_b200 import ops

pytestmark = pytest.mark.gpu
DTYPES = [torch.float32, torch.float16, torch.bfloat16]


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def normal(shape, dtype, seed):
    return torch.randn(shape, device="cuda", generator=gen(seed)).to(dtype)


def check(tokens, weight, scale, dy):
    weight = weight.detach().requires_grad_()
    y = ops.embedding(tokens, weight, scale)
    assert y.shape == (*tokens.shape, weight.shape[1]) and y.dtype == weight.dtype and y.is_contiguous()
    inside = (tokens >= 0) & (tokens < weight.shape[0])
    want = scale * weight.detach().double()[torch.where(inside, tokens, 0).long()]
    want = torch.where(inside[..., None], want, 0.0)
    bad = (tokens >= weight.shape[0])[..., None].expand_as(y)
    plain.within(torch.where(bad, 0.0, y), (want, (plain.half_step(y.dtype) + 2.0 ** -23) * want.abs() + plain.smallest(y.dtype)), "y")
    assert y[bad].isnan().all()
    (dw,) = torch.autograd.grad(y, weight, dy)
    assert dw.shape == weight.shape and dw.is_contiguous()
    value, bound = plain.embedding_gradient(tokens, dy, weight.shape[0], scale)
    plain.within(dw, (value, bound), "dw")
    assert not dw[~torch.isin(torch.arange(weight.shape[0], device="cuda"), tokens)].any()
    (again,) = torch.autograd.grad(ops.embedding(tokens, weight, scale), weight, dy)
    assert torch.equal(again, dw)


# Lengths around a warp, a chunk of 16, and the 256 warps that sort; vocabularies around the eight bits of a pass; widths around a vector, a group of threads and a CTA.
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("count,vocabulary,width", [(1, 1, 1), (1, 300, 768), (2, 2, 3), (15, 255, 8), (17, 256, 64), (31, 257, 65), (33, 65535, 7), (1000, 65536, 33), (8191, 100, 128),
                                                    (8193, 65537, 40), (20000, 70000, 16), (500, 20, 1030), (100, 50, 4100), (70001, 3, 9)])
def test_shapes(dtype, count, vocabulary, width):
    tokens = torch.randint(0, vocabulary, (count,), device="cuda", generator=gen(count))
    check(tokens, normal((vocabulary, width), dtype, 1), 1.0, normal((count, width), dtype, 2))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("how", ["same", "rising", "falling", "two", "hot", "absent", "outside", "none"])
def test_tokens(dtype, how):
    n, v, h = 5000, 1000, 72
    tokens = torch.randint(0, v, (n,), device="cuda", generator=gen(5))
    if how == "same":  # one run through all chunks
        tokens.fill_(v - 1)
    elif how in ("rising", "falling"):
        tokens = tokens.sort(descending=how == "falling").values
    elif how == "two":  # runs that end where chunks do
        tokens = torch.arange(n, device="cuda") // 2512
    elif how == "hot":
        tokens = torch.where(torch.rand(n, device="cuda", generator=gen(6)) < 0.6, 17, tokens)
    elif how == "absent":
        tokens = torch.where(torch.rand(n, device="cuda", generator=gen(6)) < 0.6, -1 - tokens, tokens)
    elif how == "outside":
        tokens = torch.where(torch.rand(n, device="cuda", generator=gen(6)) < 0.1, tokens * (1 << 40) + v, tokens)
    elif how == "none":
        tokens.fill_(-100)
    check(tokens, normal((v, h), dtype, 1), 2.5, normal((n, h), dtype, 2))


@pytest.mark.parametrize("dtype", DTYPES)
def test_strides_and_kinds(dtype):
    v, h = 300, 96
    weight, tokens, dy = normal((v, h + 8), dtype, 1), torch.randint(-2, v, (4, 50), device="cuda", generator=gen(2)), normal((4, 50, h), dtype, 3)
    check(tokens.int(), weight[:, :h], 1.0, dy)                        # rows further apart
    check(tokens, weight[:, 1:h + 1], 0.5, dy)                         # rows that do not start at 16 bytes
    check(tokens.t(), normal((h, v), dtype, 1).t(), 1.0, dy.transpose(0, 1))
    check(tokens[:, ::3], weight[::2, :h], 1.0, dy[:, ::3])
    check(tokens[:, :1].expand(4, 50), weight[:, :h], 1.0, dy)         # one token for many rows
    check(tokens, weight[:, :h], -1.0, normal((h,), dtype, 4).expand(4, 50, h))
    check(tokens, weight[:, :h], 1.0, normal((4, 50, h + 3), dtype, 4)[..., 3:])
    check(tokens[0, 0], weight[:, :h], 1.0, dy[0, 0])
    check(tokens[:0], weight[:, :h], 1.0, dy[:0])
    check(tokens, weight[:1, :h].expand(v, h), 1.0, dy)                # its gradient is that of every row


def test_infinities_stay_in_their_rows():
    tokens = torch.tensor([3, -1, 5, 3], device="cuda")
    weight, dy = torch.ones(8, 16, device="cuda"), torch.ones(4, 16, device="cuda")
    dy[1], dy[2], weight[7] = float("nan"), float("inf"), float("nan")
    y = ops.embedding(tokens, weight.requires_grad_())
    (dw,) = torch.autograd.grad(y, weight, dy)
    assert y.isfinite().all() and not y[1].any()
    assert torch.equal(dw[5], dy[2]) and torch.equal(dw[3], torch.full((16,), 2.0, device="cuda")) and not dw[[0, 1, 2, 4, 6, 7]].any()


def test_refusals():
    weight, tokens = torch.ones(8, 16, device="cuda"), torch.zeros(4, dtype=torch.long, device="cuda")
    for call in (lambda: ops.embedding(tokens.float(), weight), lambda: ops.embedding(tokens.bool(), weight), lambda: ops.embedding(tokens, weight[0]), lambda: ops.embedding(tokens, weight[:0]),
                 lambda: ops.embedding(tokens, weight[:, :0]), lambda: ops.embedding(tokens, weight.double()), lambda: ops.embedding(tokens.cpu(), weight),
                 lambda: ops.embedding(tokens, weight, scale="1"), lambda: ops.embedding(tokens, weight, scale=torch.ones((), device="cuda", requires_grad=True))):
        with pytest.raises(ValueError):
            call()
    y = ops.embedding(tokens, weight.requires_grad_())
    (dw,) = torch.autograd.grad(y.sum(), weight, create_graph=True)
    with pytest.raises(RuntimeError, match="second derivative"):
        dw.sum().backward()


def test_autocast_leaves_it_alone():
    weight = torch.randn(8, 16, device="cuda")
    with torch.autocast("cuda", dtype=torch.bfloat16):
        assert torch.equal(ops.embedding(torch.arange(8, device="cuda"), weight), weight)


def test_captured_calls_and_other_streams():
    """A lookup with its gradient in a graph, replayed with other tokens, and eager calls on another stream at the same time."""
    v, h, n = 1000, 64, 777
    weight, dy = normal((v, h), torch.bfloat16, 1).requires_grad_(), normal((n, h), torch.bfloat16, 2)
    tokens = torch.randint(0, v, (n,), device="cuda", generator=gen(3))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.autograd.grad(ops.embedding(tokens, weight, 2.0), weight, dy)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = ops.embedding(tokens, weight, 2.0)
        (dw,) = torch.autograd.grad(y, weight, dy)
    for seed in (4, 5):
        tokens.copy_(torch.randint(-1, v, (n,), device="cuda", generator=gen(seed)))
        want = ops.embedding(tokens, weight, 2.0)
        (want_dw,) = torch.autograd.grad(want, weight, dy)
        torch.cuda.synchronize()
        graph.replay()
        with torch.cuda.stream(side):
            (other,) = torch.autograd.grad(ops.embedding(tokens, weight, 2.0), weight, dy)
        torch.cuda.synchronize()
        assert torch.equal(y, want) and torch.equal(dw, want_dw) and torch.equal(other, want_dw)


def test_a_matrix_past_32_bits():
    """More than 2^31 elements, and 2^32 bytes: words at its ends."""
    v, h = (1 << 19) + 77, 4096 + 8
    assert v * h > 1 << 31
    weight = torch.zeros(v, h, dtype=torch.bfloat16, device="cuda")
    tokens = torch.tensor([v - 1, 0, v - 2, v - 1, v], device="cuda")
    weight[-2:] = normal((2, h), torch.bfloat16, 1)
    dy = normal((5, h), torch.bfloat16, 2)
    y = ops.embedding(tokens, weight.requires_grad_())
    assert torch.equal(y[0], weight[-1]) and torch.equal(y[2], weight[-2]) and not y[1].any() and y[4].isnan().all()
    (dw,) = torch.autograd.grad(y, weight, dy)
    assert torch.equal(dw[-1], (dy[0].float() + dy[3].float()).bfloat16()) and torch.equal(dw[-2], dy[2]) and torch.equal(dw[0], dy[1])
    assert not dw[1:-2].any()


def test_rows_past_32_bits():
    """More than 2^32 bytes of rows that come back; all but the last are zeros."""
    n, h, tail = (1 << 21) + 300, 1026, 50
    tokens = torch.randint(0, 64, (n,), device="cuda", generator=gen(1))
    weight = normal((64, h), torch.float16, 2).requires_grad_()
    dy = torch.zeros(n, h, dtype=torch.float16, device="cuda")
    dy[-tail:] = normal((tail, h), torch.float16, 3)
    y = ops.embedding(tokens, weight)
    assert torch.equal(y[-tail:], weight[tokens[-tail:]])
    (dw,) = torch.autograd.grad(y, weight, dy)
    plain.within(dw, plain.embedding_gradient(tokens[-tail:], dy[-tail:], 64, 1.0), "dw")


def test_a_failure_in_a_backward_pass_is_this_library_s_error():
    import ctypes
    from test_gpu_linear8 import replaced
    weight = torch.ones(8, 16, device="cuda", requires_grad=True)
    prototype = ctypes.CFUNCTYPE(ctypes.c_int, ctypes.c_void_p, ctypes.c_void_p)
    with replaced("b2_embed_backward", prototype, lambda original, *arguments: 1):
        with pytest.raises(nn.B200CclError):
            ops.embedding(torch.arange(8, device="cuda"), weight).sum().backward()
    ops.embedding(torch.arange(8, device="cuda"), weight).sum().backward()
    assert torch.equal(weight.grad, torch.ones_like(weight))
