"""The training operators and tensors that are more than memory: fake ones, wrapped ones, ones with a tangent, calls that are being traced."""
import subprocess
import sys

import pytest
import torch
import torch.utils.checkpoint

from nano_nccl_b200 import ops

pytestmark = pytest.mark.gpu

# In a process of its own: what goes wrong here ends it.
WITHOUT_MEMORY = """
import torch
from torch._subclasses.fake_tensor import FakeTensorMode
from nano_nccl_b200 import ops
p, f, w = torch.arange(5, device="cuda"), ops.rotary_frequencies(64)[0], torch.ones(64, device="cuda")
kept, dy = ops.pack8(torch.ones(5, 64, device="cuda")), torch.ones(5, 8, device="cuda")
def calls(x):
    return [lambda: ops.pack8(x), lambda: ops.gelu8(x), lambda: ops.weight_grad8(x, kept), lambda: ops.rotary(x[:, None], None, p, f),
            lambda: ops.qk_norm_rotary(x[:, None], None, w, None, p, f)]
def refused(call):
    try:
        call()
    except (RuntimeError, ValueError):
        return
    raise SystemExit("not refused")
with FakeTensorMode(allow_non_fake_inputs=True):
    fake = torch.empty(5, 64, device="cuda")
for x in (fake, torch.nn.Parameter(fake)):
    for call in calls(x):
        refused(call)
for i in range(5):
    refused(lambda: torch.func.vmap(lambda x: calls(x)[i]())(torch.ones(2, 5, 64, device="cuda")))
    refused(lambda: torch.func.grad(lambda x: (calls(x)[i](), x.sum())[1])(torch.ones(5, 64, device="cuda")))
torch.cuda.synchronize()
print("alive", float(ops.gelu8(torch.zeros(1, device="cuda"))))
"""


def test_tensors_without_memory_of_their_own():
    run = subprocess.run([sys.executable, "-c", WITHOUT_MEMORY], capture_output=True, text=True, timeout=300)
    assert run.returncode == 0 and "alive 0.0" in run.stdout, run.stderr[-2000:] + run.stdout


def arguments():
    x, w, f = torch.randn(6, 2, 64, device="cuda"), torch.ones(64, device="cuda"), ops.rotary_frequencies(64)[0]
    return x, w, f, torch.arange(6, device="cuda")


def test_forward_mode_is_refused():
    """Not dropped: an output without a tangent is a constant to whoever differentiates further."""
    x, w, f, p = arguments()
    kept = ops.pack8(x)
    with torch.autograd.forward_ad.dual_level():
        dual = lambda t: torch.autograd.forward_ad.make_dual(t, torch.ones_like(t))  # noqa: E731
        for call in (lambda: ops.pack8(dual(x)), lambda: ops.gelu8(dual(x)), lambda: ops.weight_grad8(dual(x), kept), lambda: ops.linear8(dual(x), w[None]),
                     lambda: ops.linear8(x, dual(w[None])), lambda: ops.linear8(x, w[None], dual(w[:1])), lambda: ops.rotary(dual(x), x, p, f),
                     lambda: ops.rotary(x, dual(x), p, f), lambda: ops.rotary(x, None, p, dual(f)), lambda: ops.qk_norm_rotary(dual(x), None, w, None, p, f),
                     lambda: ops.qk_norm_rotary(x, None, dual(w), None, p, f), lambda: ops.gelu8(dual(x).requires_grad_()),
                     lambda: ops.rotary(x, None, p, f, magnitude=dual(torch.ones((), device="cuda")))):
            with pytest.raises(ValueError, match="tangent|wanted"):
                call()
        # A backward pass of a gradient with a tangent (a product with the Hessian).
        leaf, weight = x.clone().requires_grad_(), w.clone()[None].requires_grad_()
        for y, by in ((ops.gelu8(leaf), leaf), (ops.rotary(leaf, None, p, f)[0], leaf), (ops.linear8(leaf, weight), weight)):
            with pytest.raises(ValueError, match="tangent"):
                torch.autograd.grad(y, by, dual(torch.ones_like(y)))


def test_gradients_that_are_not_made_are_refused():
    x, w, f, p = arguments()
    kept = ops.pack8(x)
    for call in (lambda: ops.weight_grad8(x.clone().requires_grad_(), kept), lambda: ops.rotary(x, None, p, f, magnitude=torch.ones((), requires_grad=True)),
                 lambda: ops.qk_norm_rotary(x, None, w, None, p, f, eps=torch.ones((), requires_grad=True))):
        with pytest.raises(ValueError, match="wanted"):
            call()
    with torch.no_grad():
        assert torch.equal(ops.weight_grad8(x.clone().requires_grad_(), kept)[0], ops.weight_grad8(x, kept)[0])
    assert torch.equal(ops.rotary(x, None, p, f, magnitude=torch.tensor(2.0))[0], ops.rotary(x, None, p, f, magnitude=2.0)[0])


def every_call(x, w, f, p):
    kept = ops.pack8(torch.ones(6, 2, 64, device="cuda"))
    return [lambda x: ops.pack8(x).data, lambda x: ops.unpack8(kept) * x.sum(), lambda x: ops.gelu8(x), lambda x: ops.weight_grad8(x, kept)[0],
            lambda x: ops.linear8(x, w[None]), lambda x: ops.rotary(x, None, p, f)[0], lambda x: ops.qk_norm_rotary(x, None, w, None, p, f)[0]]


@pytest.mark.filterwarnings("ignore")
def test_tracing_is_refused():
    """A trace would hold the allocation of a result and not what fills it."""
    from torch.fx.experimental.proxy_tensor import make_fx
    x, w, f, p = arguments()
    calls = every_call(x, w, f, p)
    for call in calls:
        with pytest.raises(ValueError, match="traced"):
            torch.jit.trace(call, (x,), check_trace=False)
        with pytest.raises(ValueError, match="traced"):
            make_fx(call)(x)
    del calls[1]  # (under a transformation a constant, and right)
    for call in calls:
        with pytest.raises(ValueError, match="traced|memory"):
            torch.func.vmap(call)(torch.stack([x, x]))
        with pytest.raises(ValueError, match="traced|memory"):
            torch.func.grad(lambda t: call(t).sum())(x)


@pytest.mark.filterwarnings("ignore")
def test_compilation_leaves_its_graph_for_them():
    x, w, f, p = arguments()
    calls = every_call(x, w, f, p)
    compiled = [torch.compile(call, backend="eager") for call in calls]
    for call, other in zip(calls, compiled):
        assert torch.equal(call(x), other(x))


def test_saved_tensors_may_go_elsewhere_and_be_made_again():
    """Hooks on what is saved: to the CPU and back, or made again in the backward pass."""
    x, w, f, p = arguments()
    x, w, m = x.requires_grad_(), w.requires_grad_(), torch.randn(8, 64, device="cuda", requires_grad=True)

    def step(x, w, m):
        q, _ = ops.qk_norm_rotary(x, None, w, None, p, f, keep="int8")
        return ops.gelu8(ops.linear8(ops.rotary(q, None, p, f)[0], m)).square().sum()

    want = torch.autograd.grad(step(x, w, m), (x, w, m))
    with torch.autograd.graph.save_on_cpu():
        loss = step(x, w, m)
    assert all(torch.equal(a, b) for a, b in zip(want, torch.autograd.grad(loss, (x, w, m))))
    for reentrant in (False, True):
        x.grad = w.grad = m.grad = None
        torch.utils.checkpoint.checkpoint(step, x, w, m, use_reentrant=reentrant).backward()
        assert all(torch.equal(a, b) for a, b in zip(want, (x.grad, w.grad, m.grad)))


def test_branches_of_a_captured_graph():
    """Two branches of one graph, joined in front of calls that read both: the kernels start early, and wait for both."""
    x, dy = (torch.randn(700, n, device="cuda").bfloat16() for n in (288, 320))
    q, w = torch.randn(1, 300, 4, 64, device="cuda").bfloat16(), torch.ones(64, device="cuda").bfloat16()
    f, p = ops.rotary_frequencies(64)[0], torch.arange(300, device="cuda")

    def first():
        return [ops.unpack8(ops.pack8(x)), ops.gelu8(x)]

    def second():
        return [*ops.weight_grad8(dy, ops.pack8(x * 2), bias=True), *ops.rotary(q, q, p, f), *ops.qk_norm_rotary(q, q, w, w, p, f)]

    def joined(a, b):
        return [ops.weight_grad8(dy, ops.pack8(a[1]))[0], ops.gelu8(b[0]), ops.gelu8(a[0]), *ops.qk_norm_rotary(b[2], b[5], w, w, p, f)]

    want = joined(first(), second())
    torch.cuda.synchronize()
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.graph(graph):
        main = torch.cuda.current_stream()
        side.wait_stream(main)
        with torch.cuda.stream(side):
            b = second()
        a = first()
        main.wait_stream(side)
        got = joined(a, b)
    for _ in range(10):
        for t in got:
            t.fill_(3.0)
        graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(u, v) for u, v in zip(got, want))
