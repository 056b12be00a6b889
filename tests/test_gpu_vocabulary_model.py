"""The two ends of a training step together, as TinyGPT2 calls them, alone, under the data-parallel wrapper and in a graph, against the same model with torch's own."""
import copy

import pytest
import torch

import nano_nccl_b200 as nn
from nano_nccl_b200 import ops
from nano_nccl_b200.models import TinyGPT2
from nano_nccl_b200.parallel import CclBackend, DistributedDataParallel

pytestmark = pytest.mark.gpu


def pair():
    """(the model, the same one in 64 bits with torch's own ends)"""
    torch.manual_seed(0)
    fused = TinyGPT2(vocab=500, context=40, hidden=64, layers=2, heads=4, vocabulary="fused").cuda()
    with torch.no_grad():
        fused.wte.weight.mul_(0.3)
    plain = TinyGPT2(vocab=500, context=40, hidden=64, layers=2, heads=4).cuda().double()
    plain.load_state_dict(fused.state_dict())
    return fused, plain


def batch(seed=1):
    g = torch.Generator().manual_seed(seed)
    tokens, targets = (torch.randint(0, 500, (3, 40), generator=g) for _ in range(2))
    targets[0, 30:] = -1
    return tokens.cuda(), targets.cuda()


def close(got, want, what):
    """A step in 32 bits: errors of a few hundred roundings of the largest gradient of a tensor."""
    assert (got.double() - want).abs().max() <= 2.0 ** -15 * want.abs().max(), what


def test_a_step_with_targets():
    fused, plain = pair()
    tokens, targets = batch()
    loss, want = fused(tokens, targets), plain(tokens, targets)
    assert abs(loss.double() - want) <= 2.0 ** -20 * want
    close(fused(tokens), plain(tokens), "logits")
    loss.backward()
    want.backward()
    for (name, p), q in zip(fused.named_parameters(), plain.parameters()):
        close(p.grad, q.grad, name)


def test_a_step_with_a_teacher():
    fused, plain = pair()
    tokens, _ = batch()
    g = torch.Generator().manual_seed(2)
    logits, entries = torch.randn(3, 40, 8, generator=g).cuda() * 2, torch.stack([torch.randperm(500, generator=g)[:8] for _ in range(120)]).view(3, 40, 8).cuda()
    loss = fused(tokens, teacher=(logits, entries), temperature=2.0)
    p = torch.softmax(logits.double() / 2, -1)
    log_q = torch.log_softmax(plain(tokens) / 2, -1).gather(-1, entries)
    want = 4 * (p * (p.log() - log_q)).sum(-1).mean()
    assert abs(loss.double() - want) <= 2.0 ** -19 * want
    loss.backward()
    want.backward()
    for (name, p), q in zip(fused.named_parameters(), plain.parameters()):
        close(p.grad, q.grad, name)


def test_padding_and_hooks():
    """Negative tokens are looked up as zeros and leave no gradient; the embedding is called as a module."""
    fused, _ = pair()
    tokens, targets = batch()
    seen = []
    fused.wte.register_forward_hook(lambda module, inputs, output: seen.append(output))
    tokens[0, 30:] = -1
    fused(tokens, targets).backward()
    assert len(seen) == 1 and not seen[0][0, 30:].any() and fused.wte.weight.grad.isfinite().all()


def test_under_the_data_parallel_wrapper():
    torch.cuda.set_device(0)
    comm = nn.Communicator(devices=[0], wait_timeout_ms=2000)
    fused, _ = pair()
    tokens, targets = batch()
    alone = copy.deepcopy(fused)
    alone(tokens, targets).backward()
    ddp = DistributedDataParallel(fused, CclBackend(comm))
    ddp.zero_grad()
    ddp(tokens, targets).backward()
    ddp.finish()
    torch.cuda.synchronize()
    for p, q in zip(fused.parameters(), alone.parameters()):
        assert torch.equal(p.grad, q.grad)
    comm.close()


def test_with_the_operators_in_8_bits_under_autocast():
    torch.manual_seed(0)
    fused = TinyGPT2(vocab=500, hidden=64, layers=1, heads=4, positions="rotary", checkpoints="int8", vocabulary="fused").cuda()
    tokens, targets = batch()
    with torch.autocast("cuda", dtype=torch.bfloat16):
        loss = fused(tokens, targets)
    loss.backward()
    assert loss.dtype == torch.float32 and all(p.grad is not None and p.grad.dtype == torch.float32 and p.grad.isfinite().all() for p in fused.parameters())


def test_a_captured_step():
    """Lookup, loss and both gradients of one tied matrix in a graph, replayed with other tokens."""
    weight = (0.1 * torch.randn(300, 64, device="cuda", generator=torch.Generator("cuda").manual_seed(3))).bfloat16().requires_grad_()
    tokens, targets = torch.zeros(50, dtype=torch.long, device="cuda"), torch.zeros(50, dtype=torch.long, device="cuda")

    def step():
        loss = ops.linear_cross_entropy(torch.tanh(ops.embedding(tokens, weight, 8.0)), weight, targets)
        return loss, torch.autograd.grad(loss, weight)[0]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    for seed in range(3):
        g = torch.Generator("cuda").manual_seed(seed)
        tokens.copy_(torch.randint(-1, 300, (50,), device="cuda", generator=g))
        targets.copy_(torch.randint(-1, 300, (50,), device="cuda", generator=g))
        graph.replay()
        want = step()
        assert torch.equal(captured[0], want[0]) and torch.equal(captured[1], want[1])
