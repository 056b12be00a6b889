"""Activations kept in 8 bits: the codec, GELU and the weight gradient of a projection, against plain forms in 64 bits."""
import pytest
import torch

import plain8
from nano_nccl_b200 import ops

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.float16, torch.bfloat16]


def values(shape, dtype, seed=0, scale=1.0):
    gen = torch.Generator().manual_seed(seed)
    x = torch.randn(shape, generator=gen) * scale * torch.exp(torch.randn(shape[-1], generator=gen))
    return x.clamp(-6e4, 6e4).to(dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", [(1,), (5,), (32,), (1, 1), (3, 32), (7, 31), (33, 1003), (64, 768), (2, 3, 100), (4097, 64), (5, 33)])
def test_codec(dtype, shape):
    x = values(shape, dtype, seed=len(shape))
    p = ops.pack8(x.cuda())
    got = ops.unpack8(p)
    assert got.dtype == dtype and got.shape == x.shape and got.is_contiguous()
    assert p.nbytes == x.numel() // x.shape[-1] * -(-x.shape[-1] // 32) * 33
    assert torch.equal(got.double().cpu(), plain8.kept(x))


@pytest.mark.parametrize("dtype", TYPES)
def test_codec_of_views(dtype):
    base = values((40, 200), dtype).cuda()
    for x in (base[:, :64], base[:, 3:131], base[::3, ::2], base.t(), base[1:].view(-1)[1:97], base.unsqueeze(1).expand(40, 3, 200), base[:, 32:96],
              base[:1, :96], base.view(4, 10, 200)[:, 2:7], base[:, 1:98], base[1::2, 7:40], base.view(-1)[3:3 + 61 * 128].view(61, 128)):
        assert torch.equal(ops.unpack8(ops.pack8(x)).double().cpu(), plain8.kept(x))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("columns", [64, 61])
def test_codec_at_the_ends_of_the_type(dtype, columns):
    """Zeros of both signs, smallest and largest numbers, ties, steps just below a power of two."""
    top, tiny = torch.finfo(dtype).max, torch.finfo(dtype).smallest_normal
    x = torch.zeros(10, columns)
    x[1] = -0.0
    x[2, 5], x[2, 6] = top, -top / 3
    x[3, 0], x[3, 1] = tiny, tiny / 2
    x[4, 7] = torch.finfo(dtype).eps * tiny
    x[5, :32] = torch.arange(32) * 0.5 + 56.0  # steps of one half: every other one a tie
    x[5, 0] = 127.0
    x[6, 3], x[6, 4] = 127.75, 63.5  # clamped, and a tie
    x[7, 40] = 2.0 ** -14
    x[8] = top
    x = x.to(dtype)
    assert torch.equal(ops.unpack8(ops.pack8(x.cuda())).double().cpu(), plain8.kept(x))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("columns", [96, 97])
@pytest.mark.parametrize("bad", [float("inf"), float("-inf"), float("nan")])
def test_a_block_that_is_not_finite_reads_back_as_nan(dtype, columns, bad):
    x = values((4, columns), dtype)
    x[2, 40] = bad
    got = ops.unpack8(ops.pack8(x.cuda())).cpu()
    want = plain8.kept(x)
    assert torch.isnan(got[2, 32:64]).all() and torch.isnan(want[2, 32:64]).all()
    assert torch.equal(got.double().nan_to_num(7.0), want.nan_to_num(7.0))
    dw, db = ops.weight_grad8(torch.ones(4, 8, dtype=dtype, device="cuda"), ops.pack8(x.cuda()), bias=True)
    assert torch.isnan(dw[:, 32:64]).all() and not torch.isnan(dw[:, :32]).any() and not torch.isnan(dw[:, 64:]).any()
    assert torch.equal(db, torch.full_like(db, 4.0))
    x = x.cuda().requires_grad_()
    (dx,) = torch.autograd.grad(ops.gelu8(x), x, torch.ones_like(x))
    assert torch.isnan(dx[2, 32:64]).all() and not torch.isnan(dx[1]).any()


def test_codec_of_nothing():
    for shape in ((0,), (0, 32), (5, 0), (0, 7)):
        x = torch.empty(shape, device="cuda")
        assert ops.unpack8(ops.pack8(x)).shape == shape


def test_codec_past_32_bits():
    """More than 2^32 bytes and 2^31 elements: the last rows are read and written where they lie."""
    rows, columns = (1 << 25) + 3, 65
    x = torch.zeros(rows, columns, dtype=torch.bfloat16, device="cuda")
    x[-2:] = values((2, columns), torch.bfloat16).cuda()
    got = ops.unpack8(ops.pack8(x))
    assert torch.equal(got[-2:].double().cpu(), plain8.kept(x[-2:])) and not got[:-2].any()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", [(1, 1), (3, 7), (9, 33), (5, 64), (70, 1003), (2000, 3)])
def test_outputs_at_any_address(dtype, shape):
    """The C interface takes outputs that start between multiples of 16 bytes: every element is written, and none beside them."""
    import ctypes
    import nano_nccl_b200 as nn
    lib, code = nn.load(), {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}[dtype]
    P, S, LL = ctypes.c_void_p, ctypes.c_size_t, ctypes.c_longlong
    stream = P(torch.cuda.current_stream().cuda_stream)
    x, dy = values(shape, dtype).cuda(), values(shape, dtype, seed=1).cuda()
    p = ops.pack8(x)
    n, codes = x.numel(), p.data.data_ptr()
    scales = codes + p.nbytes // 33 * 32
    leaf = x.clone().requires_grad_()
    y = ops.gelu8(leaf)
    (dx,) = torch.autograd.grad(y, leaf, dy)
    for shift in range(1, 16 // x.element_size()):
        for want, call in ((ops.unpack8(p), lambda o: lib.b2_unpack8(P(codes), P(scales), S(shape[0]), S(shape[1]), code, P(o), stream)),
                           (y, lambda o: lib.b2_gelu8_forward(P(x.data_ptr()), LL(shape[1]), S(shape[0]), S(shape[1]), code, 0, P(o), None, None, stream)),
                           (dx, lambda o: lib.b2_gelu8_backward(P(dy.data_ptr()), LL(shape[1]), P(codes), P(scales), S(shape[0]), S(shape[1]), code, 0, P(o), stream))):
            room = torch.full((n + 32,), 5.0, dtype=dtype, device="cuda")
            assert call(room.data_ptr() + shift * x.element_size()) == 0
            assert torch.equal(room[shift:shift + n], want.detach().reshape(-1)) and (room[:shift] == 5).all() and (room[shift + n:] == 5).all()


# exp(-x^2/2): the argument is rounded once, x^2/2 * 1.44 * 2^-24 <= 6.2e-6 up to |x| = 12; the polynomial and what follows are below 1e-6.
GELU_ERROR = 8e-6


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("tanh", [False, True])
@pytest.mark.parametrize("shape", [(1, 1), (7, 96), (61, 130), (3, 5, 64), (2, 1003)])
def test_gelu(dtype, tanh, shape):
    approximate = "tanh" if tanh else "none"
    base = values(shape, dtype, seed=3).clamp(-12, 12)
    x = base.cuda().requires_grad_()
    dy = values(shape, dtype, seed=4, scale=0.1).cuda()
    y = ops.gelu8(x, approximate)
    (dx,) = torch.autograd.grad(y, x, dy)
    want = plain8.gelu(base.double(), tanh)
    h = plain8.half_step(dtype)
    small = torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps + 1e-30
    # tanh: u = 0.8 (x + 0.045 x^3) is rounded three times before exp(-2u), 2|u| * 3 * 2^-24 <= 3.2e-5 where |u| <= 90; what is larger is zero.
    error = 4e-5 if tanh else GELU_ERROR
    assert ((y.double().cpu() - want).abs() <= (h + error) * want.abs() + 2 * small).all()
    v = plain8.kept(base).requires_grad_()
    (slope,) = torch.autograd.grad(plain8.gelu(v, tanh).sum(), v)
    want = dy.double().cpu() * slope
    # The two terms of the slope nearly cancel around -0.75: an error there is one of terms below 0.6, where the argument's own is below 1e-6.
    assert ((dx.double().cpu() - want).abs() <= (h + error) * want.abs() + dy.double().cpu().abs() * 4e-6 + 2 * small).all()
    with torch.no_grad():
        assert torch.equal(ops.gelu8(x, approximate), y)


def test_gelu_gradient_against_differences():
    """Inputs that 8 bits hold exactly, so that the function and the kept one are the same."""
    x = (torch.arange(-60, 61, dtype=torch.float32) / 16).repeat(4, 1)
    x = plain8.kept(x).float()
    for approximate in ("none", "tanh"):
        leaf = x.cuda().requires_grad_()
        ops.gelu8(leaf, approximate).sum().backward()
        step = 2.0 ** -8
        up, down = (ops.gelu8((x + s).cuda(), approximate).double().cpu() for s in (step, -step))
        # third derivative below 2.5: 2.5 step^2 / 6; values below 4 in 32 bits: 4 * 2^-23 / step
        assert (leaf.grad.double().cpu() - (up - down) / (2 * step)).abs().max() < 2.5 * step ** 2 / 6 + 4 * 2.0 ** -23 / step + 1e-5


def test_gelu_of_views_and_far_values():
    x = torch.tensor([[-1e30, -100.0, -0.0, 0.0, 100.0, 1e30, 3.0, float("inf")]], device="cuda")
    for approximate in ("none", "tanh"):
        y = ops.gelu8(x, approximate)
        assert torch.equal(y[0, 1:6], torch.tensor([-0.0, 0.0, 0.0, 100.0, 1e30], device="cuda")) and y[0, 7] == float("inf") and y[0, 0] == 0
        leaf = x[:, :7].clone().requires_grad_()
        ops.gelu8(leaf, approximate).sum().backward()
        assert torch.isfinite(leaf.grad).all()
    base = values((48, 96), torch.bfloat16).cuda().requires_grad_()
    for view in (lambda t: t[:, 5:40], lambda t: t.t(), lambda t: t[::2, :64]):
        x, dy = view(base), view(torch.full_like(base, 0.5))
        (dx,) = torch.autograd.grad(ops.gelu8(x), x, dy)
        (want,) = torch.autograd.grad(ops.gelu8(x.contiguous()), x, dy.contiguous())
        assert torch.equal(dx, want)


def check_weight_grad(dy, x, bias=True):
    p = ops.pack8(x)
    dw, db = ops.weight_grad8(dy, p, bias=bias)
    v = ops.unpack8(p).double().reshape(-1, x.shape[-1])
    g = dy.double().reshape(-1, dy.shape[-1])
    h = plain8.half_step(dy.dtype)
    # Every one of the T additions is off by at most 2^-23 of the sum of magnitudes so far (a cut, not a rounding).
    count = max(1, g.shape[0]) * (3 if dy.dtype == torch.float32 else 1) + 80
    want, most = g.t() @ v, g.abs().t() @ v.abs()
    tiny = torch.finfo(dy.dtype).smallest_normal
    assert dw.shape == want.shape and dw.dtype == dy.dtype
    assert ((dw.double() - want).abs() <= h * want.abs() + count * 2.0 ** -23 * most + tiny).all()
    if bias:
        assert ((db.double() - g.sum(0)).abs() <= h * g.sum(0).abs() + count * 2.0 ** -23 * g.abs().sum(0) + tiny).all()
    else:
        assert db is None
    return dw, db


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("tokens,inputs,outputs", [(1, 32, 8), (64, 256, 256), (63, 40, 24), (1, 1, 1), (130, 128, 72), (257, 300, 520), (1024, 768, 768),
                                                  (100, 33, 7), (500, 1003, 129), (2048, 64, 64), (65, 513, 257)])
def test_weight_grad(dtype, tokens, inputs, outputs):
    check_weight_grad(values((tokens, outputs), dtype, seed=5, scale=0.01).cuda(), values((tokens, inputs), dtype, seed=6).cuda())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_weight_grad_of_views(dtype):
    x = values((6, 50, 160), dtype).cuda()
    wide = values((6, 50, 400), dtype, seed=1, scale=0.1).cuda()
    for dy in (wide, wide[..., :128], wide[..., 1:98], wide[:, :, ::2], wide[:1].expand(6, 50, 400), wide[..., :1].expand(6, 50, 40)):
        check_weight_grad(dy, x, bias=False)
    check_weight_grad(wide[0, :1], x[0, :1])
    check_weight_grad(wide.permute(1, 0, 2), x.permute(1, 0, 2))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("tokens,inputs,outputs", [(26001, 700, 500), (20000, 1100, 260), (9000, 513, 4700), (16000, 64, 64), (12007, 29, 2227), (15126, 320, 61)])
def test_weight_grad_of_many_tokens(dtype, tokens, inputs, outputs):
    check_weight_grad(values((tokens, outputs), dtype, seed=5, scale=0.01).cuda(), values((tokens, inputs), dtype, seed=6).cuda())


@pytest.mark.parametrize("tokens", [1, 3, 64, 1000, 30000])
def test_weight_grad_is_exact_where_sums_are(tokens):
    """Whole numbers: every product and sum is exact, in any order, so that a term lost or taken twice shows."""
    gen = torch.Generator().manual_seed(tokens)
    for dtype in TYPES:
        x = torch.randint(-3, 4, (tokens, 200), generator=gen).to(dtype).cuda()
        x[:, ::32] = 64
        dy = torch.randint(-2, 3, (tokens, 500), generator=gen).to(dtype).cuda()
        dw, db = ops.weight_grad8(dy, ops.pack8(x), bias=True)
        want = dy.double().t() @ x.double()
        assert torch.equal(dw, want.to(dtype)) and torch.equal(db, dy.double().sum(0).to(dtype))
        for _ in range(3):
            again = ops.weight_grad8(dy, ops.pack8(x), bias=True)
            assert torch.equal(again[0], dw) and torch.equal(again[1], db)


def test_full_precision_of_float32():
    """dY with all of its 24 bits, and magnitudes over the whole range of the type: cutting it to bf16 or tf32 would show."""
    gen = torch.Generator().manual_seed(0)
    dy = torch.randn(1, 64, generator=gen) * 2.0 ** torch.randint(-60, 60, (1, 64), generator=gen)
    x = torch.full((1, 32), 1.0)
    dw, _ = ops.weight_grad8(dy.cuda(), ops.pack8(x.cuda()))
    assert ((dw.cpu().double() - dy.double().t().expand(64, 32)).abs() <= 2.0 ** -22 * dy.double().t().abs()).all()
    big = torch.tensor([[3.4e38, -3.4e38, float("inf"), float("nan")]])
    dw, db = ops.weight_grad8(big.cuda(), ops.pack8(x.cuda()), bias=True)
    assert torch.isfinite(dw[:2]).all() and (dw[2] == float("inf")).all() and torch.isnan(dw[3]).all()
    assert torch.isfinite(db[:2]).all() and db[2] == float("inf") and torch.isnan(db[3])


def test_weight_grad_of_nothing_and_repeats():
    dy, x = torch.ones(0, 24, device="cuda"), torch.ones(0, 40, device="cuda")
    dw, db = ops.weight_grad8(dy, ops.pack8(x), bias=True)
    assert dw.shape == (24, 40) and not dw.any() and db.shape == (24,) and not db.any()
    assert ops.weight_grad8(torch.ones(3, 0, device="cuda"), ops.pack8(torch.ones(3, 8, device="cuda")))[0].shape == (0, 8)
    dy, x = values((3000, 300), torch.bfloat16, scale=0.1).cuda(), values((3000, 520), torch.bfloat16).cuda()
    p = ops.pack8(x)
    first = ops.weight_grad8(dy, p, bias=True)
    for _ in range(5):
        assert all(torch.equal(a, b) for a, b in zip(first, ops.weight_grad8(dy, p, bias=True)))


@pytest.mark.parametrize("dtype", TYPES)
def test_linear(dtype):
    x, w, b = (values(s, dtype, seed=i, scale=c).cuda().requires_grad_() for i, (s, c) in enumerate([((3, 21, 96), 1.0), ((56, 96), 0.1), ((56,), 1.0)]))
    dy = values((3, 21, 56), dtype, seed=9).cuda()
    y = ops.linear8(x, w, b)
    assert torch.equal(y, torch.nn.functional.linear(x, w, b))
    dx, dw, db = torch.autograd.grad(y, (x, w, b), dy, retain_graph=True)
    assert torch.equal(dx, dy @ w)
    want = ops.weight_grad8(dy, ops.pack8(x), bias=True)
    assert torch.equal(dw, want[0]) and torch.equal(db, want[1])
    assert torch.autograd.grad(y, (b,), dy, retain_graph=True)[0].equal(db)
    assert torch.autograd.grad(ops.linear8(x, w), (w,), dy)[0].equal(dw)
    frozen = ops.linear8(x, w.detach(), b.detach())
    assert torch.autograd.grad(frozen, (x,), dy)[0].equal(dx)
    # A frozen weight: the bias's gradient needs no input. Two roundings of at most half a step each, sums of 63 terms in 32 bits beside them.
    (only_b,) = torch.autograd.grad(ops.linear8(x.detach(), w.detach(), b), (b,), dy)
    assert torch.allclose(only_b.double(), db.double(), rtol=torch.finfo(dtype).eps, atol=64 * 2.0**-24 * float(dy.abs().sum((0, 1)).max()))
    # One token without leading axes.
    dx1, dw1, db1 = torch.autograd.grad(ops.linear8(x[0, 0], w, b), (x, w, b), dy[0, 0])
    want = ops.weight_grad8(dy[0, 0], ops.pack8(x[0, 0]), bias=True)
    assert torch.equal(dx1[0, 0], dy[0, 0] @ w) and torch.equal(dw1, want[0]) and torch.equal(db1, dy[0, 0])
    # One product: exact in 32 bits where dy has 16; three parts of it added in 24 bits, cut or rounded, where it has 32.
    assert torch.allclose(dw1, torch.outer(dy[0, 0], ops.unpack8(ops.pack8(x[0, 0]))), rtol=0.0 if dtype != torch.float32 else 4 * 2.0**-23, atol=0.0)


def test_linear_under_autocast():
    x, w, b = (torch.randn(s, device="cuda", requires_grad=True) for s in ((40, 64), (32, 64), (32,)))
    with torch.autocast("cuda", dtype=torch.bfloat16):
        y = ops.linear8(x, w, b)
    assert y.dtype == torch.bfloat16
    y.float().sum().backward()
    assert x.grad.dtype == w.grad.dtype == b.grad.dtype == torch.float32 and torch.equal(b.grad, torch.full_like(b, 40.0))


def test_on_another_stream_and_in_graphs_that_live_together():
    x, dy = values((700, 288), torch.bfloat16).cuda(), values((700, 320), torch.bfloat16, seed=1, scale=0.1).cuda()

    def step():
        p = ops.pack8(x)
        return (ops.unpack8(p), *ops.weight_grad8(dy, p, bias=True))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graphs, outs = [], []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(step())
        graphs.append(g)
    for seed in range(3):
        x.copy_(values((700, 288), torch.bfloat16, seed=seed))
        streams = [torch.cuda.Stream(), torch.cuda.Stream()]
        for g, s in zip(graphs, streams):
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                g.replay()
        for s in streams:
            torch.cuda.current_stream().wait_stream(s)
        want = step()
        for got in outs:
            assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_no_second_derivative():
    x = torch.randn(8, 64, device="cuda", requires_grad=True)
    w = torch.randn(16, 64, device="cuda", requires_grad=True)
    for y, leaf in ((ops.gelu8(x), x), (ops.linear8(x, w), w)):
        (g,) = torch.autograd.grad(y.square().sum(), leaf, create_graph=True)
        with pytest.raises(RuntimeError, match="no second derivative"):
            g.sum().backward()


def test_refusals():
    x = torch.ones(4, 64, device="cuda")
    p = ops.pack8(x)
    half = ops.pack8(x.half())
    for call in (lambda: ops.pack8(x.double()), lambda: ops.pack8(x.int()), lambda: ops.pack8(x.cpu()), lambda: ops.pack8(x[0, 0]),
                 lambda: ops.unpack8(x), lambda: ops.unpack8(ops.Packed8(p.data, (4, 65), torch.float32)),
                 lambda: ops.unpack8(ops.Packed8(p.data, (4, 64), torch.float64)), lambda: ops.unpack8(ops.Packed8(p.data[1:], (4, 64), torch.float32)),
                 lambda: ops.gelu8(x, "erf"), lambda: ops.gelu8(x.double()), lambda: ops.weight_grad8(x, half), lambda: ops.weight_grad8(x[:3], p),
                 lambda: ops.weight_grad8(x.cpu(), p), lambda: ops.weight_grad8(x, x), lambda: ops.linear8(x, x.half()),
                 lambda: ops.linear8(x, torch.ones(8, 63, device="cuda")), lambda: ops.linear8(x[:, :0], torch.ones(8, 0, device="cuda")),
                 lambda: ops.pack8(torch.ones(4, 64, dtype=torch.complex64, device="cuda").conj().imag)):
        with pytest.raises(ValueError):
            call()
