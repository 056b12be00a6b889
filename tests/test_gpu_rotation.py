"""Rotation of queries and keys, alone and after the norm of each head, against plain forms in 64 bits."""
import math

import pytest
import torch

import plain8
from nano_nccl_b200 import ops

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.float16, torch.bfloat16]


def values(shape, dtype, seed=0):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(dtype)


def frequencies(rotated):
    return 10000.0 ** (-torch.arange(rotated // 2, dtype=torch.float64) * 2 / max(rotated, 1))


def angle_error(x, n, interleaved, magnitude):
    """The angle is rounded to 32 bits within half a turn (2e-7), sine and cosine are off by two units (2.4e-7), the two products and their sum by one each (1.8e-7)."""
    v = x.abs()
    out = torch.zeros_like(v)
    a, b = (slice(0, 2 * n, 2), slice(1, 2 * n, 2)) if interleaved else (slice(0, n), slice(n, 2 * n))
    out[..., a] = out[..., b] = (v[..., a] + v[..., b]) * magnitude * 7e-7
    return out


# dim, rotated, heads, kv_heads, batch, tokens
SHAPES = [(64, 64, 12, 12, 1, 1), (128, 128, 8, 2, 2, 33), (80, 40, 7, 1, 3, 21), (2, 2, 1, 1, 1, 5), (256, 256, 3, 1, 1, 9), (96, 32, 4, 4, 2, 7), (62, 30, 5, 3, 1, 17),
          (250, 6, 2, 1, 2, 3), (64, 0, 2, 2, 1, 4), (32, 16, 1, 1, 1, 300), (48, 48, 130, 1, 1, 3),
          # Halves and ends of the turning part between multiples of 16, 8 and 4 bytes; many heads of few tokens, which several warps share.
          (128, 102, 56, 8, 1, 40), (256, 190, 4, 4, 3, 20), (72, 22, 9, 3, 2, 50), (76, 76, 5, 1, 1, 130), (132, 130, 3, 2, 1, 7), (254, 254, 2, 1, 1, 6),
          (30, 30, 56, 8, 1, 31), (16, 2, 3, 3, 1, 700), (96, 24, 3, 3, 2, 90)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("shape", SHAPES)
def test_rotary(dtype, interleaved, shape):
    d, r, h, g, b, t = shape
    layout = "interleaved" if interleaved else "half"
    q, k = values((b, t, h, d), dtype).cuda().requires_grad_(), values((b, t, g, d), dtype, 1).cuda().requires_grad_()
    positions = torch.arange(t).cuda() * 37 + 11
    f = frequencies(r).cuda()
    out = ops.rotary(q, k, positions, f, layout, 1.25)
    grads = [values(o.shape, dtype, 2 + i).cuda() for i, o in enumerate(out)]
    back = torch.autograd.grad(out, (q, k), grads)
    half = plain8.half_step(dtype)
    for x, y, dy, dx in zip((q, k), out, grads, back):
        want = plain8.rotate(x.detach().double(), positions, f, interleaved, 1.25)
        assert y.shape == x.shape and y.dtype == dtype
        error = angle_error(x.detach().double(), r // 2, interleaved, 1.25)
        assert ((y.double() - want).abs() <= half * want.abs() + error + 1e-7 * (dtype == torch.float16)).all()
        assert torch.equal(y[..., r:], x[..., r:])
        want = plain8.rotate(dy.double(), -positions, f, interleaved, 1.25)
        error = angle_error(dy.double(), r // 2, interleaved, 1.25)
        assert ((dx.double() - want).abs() <= half * want.abs() + error + 1e-7 * (dtype == torch.float16)).all()


def test_far_negative_and_narrow_positions():
    q = values((2, 6, 3, 64), torch.float32).cuda()
    f = frequencies(64).cuda()
    for positions in (torch.tensor([0, 1, 999999, 12345678, 2 ** 31 - 1, -77]).cuda(), torch.tensor([[5, 4, 3, 2, 1, 0], [10 ** 9, 7, 7, 7, 8, 9]]).cuda(),
                      torch.arange(24, device="cuda").view(12, 2)[::2, 0], torch.tensor([2 ** 40, 2 ** 40 + 1, 0, 0, 0, 3]).cuda()):
        out, none = ops.rotary(q, None, positions, f)
        assert none is None
        want = plain8.rotate(q.double(), positions, f, False, 1.0)
        # position * frequency is off by 2^-52 of the turns, 2^40 / 6.3 of them at most: 4e-5 radians; below 2^32, 1e-6 of a turn's 2e-7.
        far = 3e-4 if positions.abs().max() > 2 ** 33 else 1e-6
        assert ((out.double() - want).abs() <= 2.0 ** -24 * want.abs() + angle_error(q.double(), 32, False, 1.0) + far * (q.double().abs() + 1)).all()
        if positions.max() < 2 ** 31:
            assert torch.equal(ops.rotary(None, q, positions.int(), f)[1], out)


def test_views_layouts_and_three_axes():
    base = values((2, 9, 20 * 64), torch.bfloat16).cuda()
    f = frequencies(64).cuda()
    positions = torch.arange(9, device="cuda")
    q, k = base[..., :12 * 64].view(2, 9, 12, 64), base[..., 12 * 64:16 * 64].view(2, 9, 4, 64)
    want = ops.rotary(q.contiguous(), k.contiguous(), positions, f)
    same = lambda got: all(torch.equal(a, b) for a, b in zip(got, want))  # noqa: E731
    assert same(ops.rotary(q, k, positions, f))
    by_heads = [t.transpose(1, 2).contiguous().transpose(1, 2) for t in (q, k)]
    assert same(ops.rotary(*by_heads, positions, f))
    padded = [torch.nn.functional.pad(t, (1, 2))[..., 1:-2] for t in (q, k)]  # rows at odd addresses
    assert same(ops.rotary(*padded, positions, f))
    last = [t.transpose(2, 3).contiguous().transpose(2, 3) for t in (q, k)]  # the last axis has gaps
    assert same(ops.rotary(*last, positions, f))
    assert same([torch.stack(o) for o in zip(*(ops.rotary(q[i], k[i], positions, f) for i in range(2)))])
    leaf = q.detach().requires_grad_()
    out, _ = ops.rotary(leaf, None, positions, f)
    out.sum().backward()  # a gradient without memory of its own
    assert torch.equal(leaf.grad, ops.rotary(torch.ones_like(q), None, -positions, f)[0])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("d,r", [(128, 102), (128, 72), (64, 22), (72, 22), (76, 38), (30, 14), (64, 0), (30, 0), (76, 0)])
def test_what_does_not_turn_stays_as_it_is(dtype, interleaved, d, r):
    """To the last bit, whatever stands beside it: infinities, NaN, zeros with signs."""
    x = values((1, 40, 3, d), dtype).cuda()
    x[0, :10] = float("inf")
    x[0, 10:20, :, :r] = float("nan")
    x[0, 20:30, :, ::2] = float("-inf")
    x[0, 30:] = -0.0
    y, _ = ops.rotary(x, None, torch.arange(40).cuda(), frequencies(r).cuda(), "interleaved" if interleaved else "half")
    as_bits = torch.int32 if dtype == torch.float32 else torch.int16
    assert torch.equal(y[..., r:].contiguous().view(as_bits), x[..., r:].contiguous().view(as_bits))
    assert y[0, 10:20, :, :r].isnan().all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("keep", ["int8", None])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("shape", SHAPES)
def test_norm(dtype, keep, interleaved, shape):
    d, r, h, g, b, t = shape
    layout = "interleaved" if interleaved else "half"
    q, k = ((3 * values((b, t, n, d), torch.float32, i)).to(dtype).cuda().requires_grad_() for i, n in enumerate((h, g)))
    w = [(1 + 0.1 * values((d,), torch.float32, 5 + i)).to(dtype).cuda().requires_grad_() for i in range(2)]
    positions = torch.arange(t).cuda() * 13 + 5
    f = frequencies(r).cuda()
    eps, magnitude = 1e-5, 0.75
    out = ops.qk_norm_rotary(q, k, *w, positions, f, layout, magnitude, eps, keep)
    grads = [values(o.shape, dtype, 2 + i).cuda() for i, o in enumerate(out)]
    back = torch.autograd.grad(out, (q, k, *w), grads)
    half = plain8.half_step(dtype)
    tiny = 2.0 ** -24 if dtype == torch.float16 else 1e-30
    for i, x in enumerate((q, k)):
        weight = w[i].detach().double()

        def forward(v, u):
            return plain8.rotate(v / torch.sqrt((v * v).mean(-1, keepdim=True) + eps) * u, positions, f, interleaved, magnitude)

        v = x.detach().double()
        n = v / torch.sqrt((v * v).mean(-1, keepdim=True) + eps) * weight
        want = forward(v, weight)
        # The sum of d squares is off by (d / 32 + 8) roundings at most, its root by half of that, and four more follow.
        sums = (d / 64 + 10) * 2.0 ** -24
        assert ((out[i].double() - want).abs() <= half * want.abs() + angle_error(n, r // 2, interleaved, magnitude) + 2 * sums * n.abs() + sums * magnitude * n.abs().amax(-1, keepdim=True) + tiny).all()
        v = (plain8.kept(x, d).cuda() if keep else v).requires_grad_()
        u = weight.clone().requires_grad_()
        dy = grads[i].double()
        dx, dw = torch.autograd.grad(forward(v, u), (v, u), dy)
        rstd = 1 / torch.sqrt((v * v).mean(-1, keepdim=True) + eps)
        gr = plain8.rotate(dy, -positions, f, interleaved, magnitude)
        gw, norm = (gr * weight).abs(), (v * rstd).abs()
        error = 1e-6 * rstd * dy.abs().amax(-1, keepdim=True) * weight.abs().amax() + 4 * sums * rstd * (gw + norm * (gw * norm).mean(-1, keepdim=True))
        assert ((back[i].double() - dx).abs() <= half * dx.abs() + error + tiny).all()
        # b * t * heads terms, added by 8 to 256 rows at a time, then by CTA: as many roundings as terms at most, and the error of each term.
        terms = (gr.abs() * norm).sum((0, 1, 2)) + 2e-6 * (dy.abs().amax(-1, keepdim=True) * norm).sum((0, 1, 2)) / 2.0 ** -20
        count = b * t * (h, g)[i] + 40
        assert ((back[2 + i].double() - dw).abs() <= half * dw.abs() + (count * 2.0 ** -24 + 4 * sums) * (gr.abs() * norm).sum((0, 1, 2)) + 2.0 ** -20 * terms + tiny).all()
    with torch.no_grad():
        again = ops.qk_norm_rotary(q, k, *w, positions, f, layout, magnitude, eps, keep)
    assert all(torch.equal(a, o) for a, o in zip(again, out))


def test_norm_gradient_against_differences():
    """Heads that 8 bits hold exactly, and a fixed direction: the slope of the summed output along it."""
    gen = torch.Generator().manual_seed(1)
    x = torch.randint(-127, 128, (4, 3, 64), generator=gen).float() / 64
    x[..., 0] = 127 / 64
    way, dy, w = (torch.randn(s, generator=gen) for s in ((4, 3, 64), (4, 3, 64), (64,)))
    positions, f = torch.arange(4).cuda(), frequencies(64).cuda()
    leaf, weight = x.cuda().requires_grad_(), w.cuda().requires_grad_()
    out, _ = ops.qk_norm_rotary(leaf, None, weight, None, positions, f)
    dx, dw = torch.autograd.grad(out, (leaf, weight), dy.cuda())
    step = 2.0 ** -7

    def total(v, u):
        return (ops.qk_norm_rotary(v.cuda(), None, u.cuda(), None, positions, f)[0].double().cpu() * dy.double()).sum().item()

    slope = (total(x + step * way, w) - total(x - step * way, w)) / (2 * step)
    assert abs(slope - (dx.cpu().double() * way.double()).sum().item()) < 0.02 * way.norm().item()
    slope = (total(x, w + step * way[0, 0]) - total(x, w - step * way[0, 0])) / (2 * step)  # linear in the weight
    assert abs(slope - (dw.cpu().double() * way[0, 0].double()).sum().item()) < 1e-2


def test_norm_sides_and_kept_bytes():
    b, t, d = 2, 50, 64
    q, k = values((b, t, 8, d), torch.bfloat16).cuda().requires_grad_(), values((b, t, 2, d), torch.bfloat16, 1).cuda().requires_grad_()
    w = [torch.ones(d, dtype=torch.bfloat16, device="cuda").requires_grad_() for _ in range(2)]
    positions, f = torch.arange(t).cuda(), frequencies(d).cuda()
    dq, dk = values(q.shape, torch.bfloat16, 3).cuda(), values(k.shape, torch.bfloat16, 4).cuda()
    both = torch.autograd.grad(ops.qk_norm_rotary(q, k, *w, positions, f), (q, k, *w), (dq, dk))
    out = ops.qk_norm_rotary(q, k, *w, positions, f)
    only_k = torch.autograd.grad(out[1], (k, w[1]), dk, retain_graph=True)  # the other output is not used
    assert torch.equal(only_k[0], both[1])
    alone = torch.autograd.grad(ops.qk_norm_rotary(q, None, w[0], None, positions, f)[0], (q, w[0]), dq)
    assert torch.equal(alone[0], both[0])
    # A row of zeros has a gradient (eps holds it), one that is not finite has NaN, and neither touches its neighbours.
    with torch.no_grad():
        q[0, 3, 1] = 0
        q[1, 7, 2, 5] = float("inf")
    dx = torch.autograd.grad(ops.qk_norm_rotary(q, k, *w, positions, f)[0], (q,), dq)[0]
    assert torch.isfinite(dx[0, 3, 1]).all() and torch.isnan(dx[1, 7, 2]).all()
    keep = torch.ones(b, t, 8, dtype=torch.bool)
    keep[0, 3, 1] = keep[1, 7, 2] = False
    assert torch.equal(dx[keep.cuda()], both[0][keep.cuda()])


def test_nothing_repeats_streams_and_graphs():
    w = [torch.ones(64, device="cuda").requires_grad_() for _ in range(2)]
    f = frequencies(64).cuda()
    q, k = torch.empty(0, 4, 64, device="cuda", requires_grad=True), torch.empty(0, 2, 64, device="cuda", requires_grad=True)
    out = ops.qk_norm_rotary(q, k, *w, torch.arange(0, device="cuda"), f)
    grads = torch.autograd.grad(out, (q, k, *w), [torch.empty_like(o) for o in out])
    assert grads[0].shape == q.shape and not grads[2].any() and not grads[3].any()
    q, k = values((1, 3000, 8, 64), torch.bfloat16).cuda().requires_grad_(), values((1, 3000, 8, 64), torch.bfloat16, 1).cuda().requires_grad_()
    w = [torch.ones(64, dtype=torch.bfloat16, device="cuda").requires_grad_() for _ in range(2)]
    positions = torch.arange(3000, device="cuda")
    dy = [values(t.shape, torch.bfloat16, 5 + i).cuda() for i, t in enumerate((q, k))]

    def step():
        return torch.autograd.grad(ops.qk_norm_rotary(q, k, *w, positions, f), (q, k, *w), dy)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        first = [g.clone() for g in step()]
    torch.cuda.current_stream().wait_stream(side)
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(first, step()))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    for g in captured:
        g.zero_()
    graph.replay()
    assert all(torch.equal(a, b) for a, b in zip(first, captured))


def test_refusals():
    q, w = torch.ones(5, 3, 64, device="cuda"), torch.ones(64, device="cuda")
    p, f = torch.arange(5, device="cuda"), frequencies(64).cuda()
    for call in (lambda: ops.rotary(None, None, p, f), lambda: ops.rotary(q.cpu(), None, p, f), lambda: ops.rotary(q, q.half(), p, f),
                 lambda: ops.rotary(q, q[:4], p, f), lambda: ops.rotary(q, None, p[:4], f), lambda: ops.rotary(q, None, p.float(), f),
                 lambda: ops.rotary(q, None, p, f.float()), lambda: ops.rotary(q, None, p, frequencies(66).cuda()), lambda: ops.rotary(q[..., :63], None, p, f[:8]),
                 lambda: ops.rotary(q, None, p, f, "quarter"), lambda: ops.rotary(q[0], None, p, f), lambda: ops.rotary(q.double(), None, p, f),
                 lambda: ops.rotary(torch.ones(5, 1, 258, device="cuda"), None, p, f), lambda: ops.rotary(q, None, p, f[::2]),
                 lambda: ops.rotary(q[None], None, torch.stack([p, p]), f), lambda: ops.rotary(q[:, :0], None, p, f),
                 lambda: ops.qk_norm_rotary(q, None, None, None, p, f), lambda: ops.qk_norm_rotary(q, None, w[:32], None, p, f),
                 lambda: ops.qk_norm_rotary(q, None, w.half(), None, p, f), lambda: ops.qk_norm_rotary(q, None, w, None, p, f, keep="fp8"),
                 lambda: ops.qk_norm_rotary(q, None, w, None, p, f, eps=-1.0), lambda: ops.qk_norm_rotary(q, q, w, None, p, f),
                 lambda: ops.rotary(q, None, p, f.clone().requires_grad_()), lambda: ops.qk_norm_rotary(q, None, w, None, p, f.clone().requires_grad_())):
        with pytest.raises(ValueError):
            call()


@pytest.mark.parametrize("keep", [None, "int8"])
def test_norm_under_autocast(keep):
    q, k = (torch.randn(2, 9, h, 64, device="cuda", dtype=torch.bfloat16) for h in (4, 2))
    w = [torch.linspace(0.5, 1.5, 64, device="cuda", requires_grad=True) for _ in range(2)]
    p, f = torch.arange(9, device="cuda"), frequencies(64).cuda()
    with torch.autocast("cuda", dtype=torch.bfloat16):
        got = ops.qk_norm_rotary(q, k, *w, p, f, keep=keep)
    narrow = [v.detach().bfloat16().requires_grad_() for v in w]
    want = ops.qk_norm_rotary(q, k, *narrow, p, f, keep=keep)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    for grads in zip(torch.autograd.grad([v.float().square().sum() for v in got], w), torch.autograd.grad([v.float().square().sum() for v in want], narrow)):
        assert grads[0].dtype == torch.float32 and torch.equal(grads[0], grads[1].float())


def test_scaled_frequencies():
    base, one = ops.rotary_frequencies(64, device="cpu")
    assert torch.allclose(base, frequencies(64), rtol=1e-14, atol=0) and one == 1.0
    assert torch.allclose(ops.rotary_frequencies(64, scaling="linear", factor=4.0, device="cpu")[0] * 4, base, rtol=1e-14, atol=0)
    ntk, _ = ops.rotary_frequencies(64, scaling="ntk", factor=4.0, device="cpu")
    assert math.isclose(ntk[0], base[0]) and math.isclose(ntk[-1], base[-1] / 4, rel_tol=1e-12)
    yarn, m = ops.rotary_frequencies(64, scaling="yarn", factor=4.0, context=4096, device="cpu")
    turns = base * 4096 / (2 * math.pi)
    assert torch.equal(yarn[turns > 64], base[turns > 64]) and torch.allclose(yarn[turns < 0.5], base[turns < 0.5] / 4) and m == 0.1 * math.log(4) + 1
    assert ((yarn <= base) & (yarn >= base / 4 * (1 - 1e-12))).all()
