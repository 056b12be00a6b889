"""The training operators at their far ends: tensors past 32 bits, calls of several threads, a first call inside a capture."""
import subprocess
import sys
import threading

import pytest
import torch

from nano_nccl_b200 import ops

pytestmark = pytest.mark.gpu


def values(shape, seed, scale=1.0):
    return (torch.randn(shape, generator=torch.Generator().manual_seed(seed)) * scale).bfloat16().cuda()


@pytest.mark.parametrize("columns", [2047, 2048])
def test_gelu(columns):
    """More than 2^32 elements: the last rows are those of a call of their own."""
    rows, tail = (1 << 21) + 5000, 70
    assert rows * columns > 1 << 32
    x, dy = torch.zeros(rows, columns, dtype=torch.bfloat16, device="cuda"), torch.zeros(rows, columns, dtype=torch.bfloat16, device="cuda")
    x[-tail:], dy[-tail:] = values((tail, columns), 0), values((tail, columns), 1)
    x.requires_grad_()
    small = x[-tail:].detach().clone().requires_grad_()
    y, want = ops.gelu8(x), ops.gelu8(small)
    assert torch.equal(y[-tail:], want) and not y[:-tail].any()
    del y
    (dx,) = torch.autograd.grad(ops.gelu8(x), x, dy)
    assert torch.equal(dx[-tail:], torch.autograd.grad(want, small, dy[-tail:])[0]) and not dx[:-tail].any()


@pytest.mark.parametrize("keep", [None, "int8"])
def test_head_norms(keep):
    """Queries of more than 2^31 elements."""
    tokens, tail = (1 << 20) + 3, 37
    f, _ = ops.rotary_frequencies(128)
    positions = torch.arange(tokens, device="cuda")
    q, k = (torch.zeros(tokens, heads, 128, dtype=torch.bfloat16, device="cuda") for heads in (24, 2))
    dy = [torch.zeros_like(q), torch.zeros_like(k)]
    for i, t in enumerate((q, k, *dy)):
        t[-tail:] = values(t[-tail:].shape, i)
    w = [values((128,), 8).requires_grad_(), values((128,), 9).requires_grad_()]
    small = [t[-tail:].clone().requires_grad_() for t in (q, k)]
    want = ops.qk_norm_rotary(*small, *w, positions[-tail:], f, keep=keep)
    want_grads = torch.autograd.grad(want, (*small, *w), [t[-tail:] for t in dy])
    got = ops.qk_norm_rotary(q.requires_grad_(), k.requires_grad_(), *w, positions, f, keep=keep)
    assert all(torch.equal(a[-tail:], b) and not a[:-tail].any() for a, b in zip(got, want))
    grads = torch.autograd.grad(got, (q, k, *w), dy)
    assert all(torch.equal(a[-tail:], b) and not a[:-tail].any() for a, b in zip(grads[:2], want_grads[:2]))
    # The same 37 * heads products, added in another order in 32 bits, then rounded: a step, and 900 * 2^-24 of sums of magnitudes (below 1e3 here).
    for a, b in zip(grads[2:], want_grads[2:]):
        assert torch.allclose(a.double(), b.double(), rtol=2.0**-7, atol=0.06)


@pytest.mark.parametrize("outputs", [2056, 2051])
def test_weight_grad_of_long_sums(outputs):
    """dY of more than 2^32 elements, read as it lies and copied. All but the last tokens are zeros."""
    tokens, tail = (1 << 21) + 10000, 100
    assert tokens * outputs > 1 << 32
    dy, x = torch.zeros(tokens, outputs, dtype=torch.bfloat16, device="cuda"), torch.zeros(tokens, 96, dtype=torch.bfloat16, device="cuda")
    dy[-tail:], x[-tail:] = values((tail, outputs), 0), values((tail, 96), 1)
    dw, db = ops.weight_grad8(dy, ops.pack8(x), bias=True)
    g, v = dy[-tail:].double(), ops.unpack8(ops.pack8(x[-tail:])).double()
    # 100 additions, each off by at most 2^-23 of the magnitudes so far, and a rounding to 8 bits.
    for got, want, most in ((dw, g.t() @ v, g.abs().t() @ v.abs()), (db, g.sum(0), g.abs().sum(0))):
        assert ((got.double() - want).abs() <= 2.0**-8 * want.abs() + 200 * 2.0**-23 * most).all()


def test_weight_grad_of_many_tiles():
    """A result of more than 2^32 elements."""
    n, tokens = 65600, 70
    dy, x = values((tokens, n), 0), values((tokens, n), 1)
    p = ops.pack8(x)
    dw, _ = ops.weight_grad8(dy, p)
    v = ops.unpack8(p)
    for rows in (slice(0, 300), slice(40000, 40300), slice(n - 300, n)):
        for columns in (slice(0, 300), slice(n - 300, n)):
            g, u = dy[:, rows].double(), v[:, columns].double()
            want = g.t() @ u
            assert ((dw[rows, columns].double() - want).abs() <= 2.0**-8 * want.abs() + 200 * 2.0**-23 * (g.abs().t() @ u.abs())).all()


def test_calls_of_several_threads():
    inputs = [(values((700 + 64 * i, 288), i), values((700 + 64 * i, 320), 10 + i, 0.1)) for i in range(4)]
    want = [ops.weight_grad8(dy, ops.pack8(x), bias=True) for x, dy in inputs]
    torch.cuda.synchronize()
    got, failures = [None] * 4, []

    def work(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(20):
                    got[i] = ops.weight_grad8(inputs[i][1], ops.pack8(inputs[i][0]), bias=True)
                torch.cuda.current_stream().synchronize()
            for bad in (inputs[i][0].cpu(), inputs[i][0].double()):
                with pytest.raises(ValueError):
                    ops.pack8(bad)
        except BaseException as e:  # noqa: B036 (a thread's failure is the test's)
            failures.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failures
    assert all(torch.equal(a, b) for g, w in zip(got, want) for a, b in zip(g, w))


FIRST_CALL_CAPTURED = """
import torch
from nano_nccl_b200 import ops
x = torch.randn(300, 288, device="cuda").bfloat16()
dy = torch.randn(300, 320, device="cuda").bfloat16()
q, w = torch.randn(1, 9, 4, 64, device="cuda").bfloat16(), torch.ones(64, device="cuda").bfloat16()
f, p = ops.rotary_frequencies(64)[0], torch.arange(9, device="cuda")
def step():
    kept = ops.pack8(x)
    return [ops.unpack8(kept), ops.gelu8(x), *ops.weight_grad8(dy, kept, bias=True), *ops.rotary(q, q, p, f), *ops.qk_norm_rotary(q, q, w, w, p, f)]
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    captured = step()
graph.replay()
torch.cuda.synchronize()
assert all(torch.equal(a, b) for a, b in zip(captured, step()))
print("the same")
"""


def test_a_first_call_inside_a_capture():
    run = subprocess.run([sys.executable, "-c", FIRST_CALL_CAPTURED], capture_output=True, text=True, timeout=300)
    assert run.returncode == 0 and "the same" in run.stdout, run.stderr[-2000:]
