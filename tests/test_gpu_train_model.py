"""The training operators together, as TinyGPT2 calls them under the data-parallel wrapper, against the same model in 64 bits
whose backward pass sees the same 8-bit values."""
import copy

import pytest
import torch

import nano_nccl_b200 as nn
import plain8
from nano_nccl_b200 import ops
from nano_nccl_b200.models import TinyGPT2
from nano_nccl_b200.parallel import CclBackend, DistributedDataParallel

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def comm():
    torch.cuda.set_device(0)
    c = nn.Communicator(devices=[0], wait_timeout_ms=2000)
    yield c
    c.close()


def kept32(x, block=32):
    """What the 8-bit form of a float32 value stands for."""
    return plain8.kept(x.detach().float(), block).to(x.device)


class KeptGelu(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x):
        ctx.save_for_backward(kept32(x))
        return plain8.gelu(x, False)

    @staticmethod
    def backward(ctx, dy):
        with torch.enable_grad():
            v = ctx.saved_tensors[0].requires_grad_()
            return torch.autograd.grad(plain8.gelu(v, False), v, dy)[0]


class KeptLinear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w, b):
        ctx.save_for_backward(kept32(x), w)
        return x @ w.t() + b

    @staticmethod
    def backward(ctx, dy):
        v, w = ctx.saved_tensors
        flat = dy.reshape(-1, dy.shape[-1])
        return dy @ w, flat.t() @ v.reshape(-1, v.shape[-1]), flat.sum(0)


class KeptNorm(torch.autograd.Function):
    @staticmethod
    def norm(x, w):
        return x * torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-6) * w

    @staticmethod
    def forward(ctx, x, w):
        ctx.save_for_backward(kept32(x, x.shape[-1]), w)
        return KeptNorm.norm(x, w)

    @staticmethod
    def backward(ctx, dy):
        with torch.enable_grad():
            v, w = (t.detach().requires_grad_() for t in ctx.saved_tensors)
            return torch.autograd.grad(KeptNorm.norm(v, w), (v, w), dy)


def plain_forward(model, tokens):
    """`model` is in 64 bits; its options are those with rotary positions, head norms and 8-bit checkpoints."""
    x = model.wte(tokens)
    linear = lambda x, layer: KeptLinear.apply(x, layer.weight, layer.bias)  # noqa: E731
    for block in model.blocks:
        a, (b, t, hidden) = block.attn, x.shape
        q, k, v = (p.view(b, t, a.heads, -1) for p in linear(block.ln_1(x), a.c_attn).split(hidden, -1))
        positions, f = torch.arange(t, device=x.device), a.frequencies(x.device)
        q, k = (plain8.rotate(KeptNorm.apply(p, w), positions, f, False, 1.0) for p, w in ((q, a.q_norm), (k, a.k_norm)))
        scores = torch.einsum("bqhd,bkhd->bhqk", q, k) / (hidden // a.heads) ** 0.5
        y = torch.einsum("bhqk,bkhd->bqhd", scores.softmax(-1), v).reshape(b, t, hidden)
        x = x + linear(y, a.c_proj)
        x = x + linear(KeptGelu.apply(linear(block.ln_2(x), block.mlp[0])), block.mlp[2])
    return model.ln_f(x) @ model.wte.weight.t()


def test_a_data_parallel_step(comm):
    torch.manual_seed(0)
    model = TinyGPT2(vocab=96, context=32, hidden=96, layers=2, heads=3, positions="rotary", qk_norm=True, checkpoints="int8").cuda()
    wide = copy.deepcopy(model).double()
    tokens = torch.randint(0, 96, (3, 29), device="cuda")
    ddp = DistributedDataParallel(model, CclBackend(comm), bucket_bytes=64 << 10)
    logits = ddp(tokens)
    logits.logsumexp(-1).mean().backward()
    ddp.finish()
    want = plain_forward(wide, tokens)
    want.logsumexp(-1).mean().backward()
    torch.cuda.synchronize()
    comm.check_async_error()
    # A forward pass in 32 bits: sums of up to 384 terms, twice two layers, below 2^-24 * 400 * 8 of the logits' size.
    assert (logits.double() - want).abs().max() < 2e-4 * want.abs().max()
    # Gradients: an activation that is 1e-6 off falls on the other side of a rounding in one of 1e4 cases (a step is at least 1/128 of the
    # block's largest), and is then off by a step: 1e-2 * 1e-2 of the gradient's norm, and no more than ten times that after two layers.
    for (name, p), q in zip(model.named_parameters(), wide.parameters()):
        assert (p.grad.double() - q.grad).norm() <= 1e-3 * q.grad.norm() + 1e-9, name


@pytest.mark.parametrize("options", [dict(positions="rotary"), dict(qk_norm=True), dict(checkpoints="int8"), dict(positions="rotary", qk_norm=True, checkpoints="int8")])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_a_captured_step_repeats_the_eager_one(options, dtype):
    torch.manual_seed(1)
    model = TinyGPT2(vocab=64, context=16, hidden=64, layers=2, heads=2, **options).cuda().to(dtype)
    tokens = torch.randint(0, 64, (4, 16), device="cuda")
    for p in model.parameters():
        p.grad = torch.zeros_like(p)

    def step():
        for p in model.parameters():
            p.grad.zero_()
        loss = model(tokens).float().logsumexp(-1).mean()
        loss.backward()
        return loss.detach()

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step()
    torch.cuda.current_stream().wait_stream(side)
    eager = step()
    want = [p.grad.clone() for p in model.parameters()]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    for p in model.parameters():
        p.grad.fill_(7.0)
    graph.replay()
    torch.cuda.synchronize()
    # (Embedding gradients are torch's, summed by atomics.)
    for (name, p), w in zip(model.named_parameters(), want):
        assert torch.equal(p.grad, w) if "wte" not in name and "wpe" not in name else torch.allclose(p.grad, w, rtol=2e-2, atol=1e-5), name
    assert torch.equal(captured, eager)


def test_a_step_under_autocast():
    torch.manual_seed(2)
    model = TinyGPT2(vocab=64, context=16, hidden=64, layers=2, heads=2, positions="rotary", qk_norm=True, checkpoints="int8").cuda()
    tokens = torch.randint(0, 64, (4, 16), device="cuda")
    with torch.autocast("cuda", dtype=torch.bfloat16):
        loss = model(tokens).float().logsumexp(-1).mean()
    loss.backward()
    for name, p in model.named_parameters():
        assert p.grad.dtype == torch.float32 and p.grad.isfinite().all() and p.grad.any(), name


def test_what_a_step_keeps():
    """The point of it: 33 bytes for 32 elements instead of 64 or 128."""
    def kept(f, *leaves):
        torch.cuda.synchronize()
        before = torch.cuda.memory_allocated()
        y = f(*leaves)
        return torch.cuda.memory_allocated() - before - y.numel() * y.element_size()

    x = torch.randn(4096, 2048, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    assert kept(lambda t: ops.gelu8(t * 1.0), x) <= 4096 * 2048 * 33 / 32 * 1.01
    w = torch.randn(512, 2048, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    assert kept(lambda t: ops.linear8(t * 1.0, w), x) <= 4096 * 2048 * 33 / 32 * 1.01
