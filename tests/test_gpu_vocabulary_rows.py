"""Losses over a vocabulary: what one row is must not reach another's loss or gradient, and the ways that a call may take are each held to what that way may lose."""
import copy
import ctypes

import pytest
import torch

import nano_nccl_b200 as nn
import plain_vocabulary as plain
from nano_nccl_b200 import ops
from nano_nccl_b200.models import TinyGPT2
from nano_nccl_b200.parallel import CclBackend, DistributedDataParallel
from test_cpu_vocabulary_ops import LL, VocabularyLoss
from test_gpu_linear8 import replaced
from test_gpu_vocabulary_loss import DTYPES, cross_entropy, distillation, gen, inputs, made_with_the_loss, normal, run, teacher

pytestmark = pytest.mark.gpu


def each_row_alone(out, x, w, targets, dloss, rows, logits=None, temperature=1.0):
    """The loss and the gradient of x of some rows, each against the formula of that row alone: its bound knows nothing of the others."""
    for t in rows:
        part = slice(t, t + 1)
        want = plain.losses(x[part], w, targets[part], None if logits is None else logits[part], temperature, "none", dloss[part])
        for name in ("loss", "dx"):
            plain.within(out[name][part], want[name], f"{name} of row {t}")


# ---- float32: rows of very different sizes ---------------------------------------------------------------

@pytest.mark.parametrize("size", [1e10, 1e30])
@pytest.mark.parametrize("reduction", ["none", "mean"])
def test_what_a_padded_row_holds_does_not_matter(size, reduction):
    x, w, t = inputs(100, 700, 72, torch.float32)
    padded = t < 0
    dloss = torch.rand(100, device="cuda", generator=gen(5)) + 0.5 if reduction == "none" else torch.tensor(0.75, device="cuda")
    want = run(cross_entropy(t, reduction), torch.where(padded[:, None], 0.0, x), w, dloss)
    got = run(cross_entropy(t, reduction), torch.where(padded[:, None], size, x), w, dloss)
    assert all(torch.equal(got[name], want[name]) for name in want)
    counted = ~padded
    exact = plain.losses(x[counted], w, t[counted], reduction=reduction, dloss=dloss[counted] if reduction == "none" else dloss)
    plain.within(got["loss"][counted] if reduction == "none" else got["loss"], exact["loss"], "loss")
    plain.within(got["dx"][counted], exact["dx"], "dx")
    plain.within(got["dw"], exact["dw"], "dw")
    logits, tokens = teacher(100, 5, 700, torch.float32)
    tokens[padded] = -1
    call = distillation(logits, tokens, 2.0, reduction)
    want, got = run(call, torch.where(padded[:, None], 0.0, x), w, dloss), run(call, torch.where(padded[:, None], size, x), w, dloss)
    assert all(torch.equal(got[name], want[name]) for name in want)


def test_rows_of_any_size_have_their_own_loss_and_gradient():
    """Rows of 1e-12 to 1e10, some of zeros: the logits and the gradient of each lose what its own elements lose."""
    rows = 60
    x, w, t = inputs(rows, 700, 72, torch.float32)
    t = t.clamp(min=0)
    x = x * 10.0 ** torch.linspace(-12, 10, rows, device="cuda")[:, None]
    x[7] = 0.0
    dloss = torch.rand(rows, device="cuda", generator=gen(5)) + 0.5
    out = run(cross_entropy(t, "none"), x, w, dloss)
    each_row_alone(out, x, w, t, dloss, range(rows))
    plain.within(out["dw"], plain.losses(x, w, t, reduction="none", dloss=dloss)["dw"], "dw")
    logits, tokens = teacher(rows, 5, 700, torch.float32)
    out = run(distillation(logits, tokens, 2.0, "none"), x, w, dloss)
    each_row_alone(out, x, w, tokens, dloss, range(rows), logits, 2.0)


def test_a_row_s_own_infinities_stay_its_own():
    x, w, t = inputs(60, 300, 64, torch.float32)
    t = t.clamp(min=0)
    spoilt = x.clone()
    spoilt[3, 5], spoilt[9, 0] = float("inf"), float("nan")
    dloss = torch.ones(60, device="cuda")
    got, want = run(cross_entropy(t, "none"), spoilt, w, dloss), run(cross_entropy(t, "none"), x, w, dloss)
    others = torch.ones(60, dtype=torch.bool, device="cuda")
    others[[3, 9]] = False
    assert torch.equal(got["loss"][others], want["loss"][others]) and torch.equal(got["dx"][others], want["dx"][others])
    assert not got["loss"][~others].isfinite().any() and not got["dx"][~others].isfinite().any()


# ---- what comes back to rows that are weighted one by one ------------------------------------------------

@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("frozen", [False, True])
def test_a_weight_that_is_no_number_stays_in_its_row(dtype, frozen):
    x, w, t = inputs(80, 700, 72, dtype)
    t = t.clamp(min=0)
    dloss = torch.rand(80, device="cuda", generator=gen(5)) + 0.5
    spoilt, without = dloss.clone(), dloss.clone()
    spoilt[5], spoilt[9], spoilt[70] = float("inf"), float("nan"), -float("inf")
    without[[5, 9, 70]] = 0.0
    logits, tokens = teacher(80, 5, 700, dtype)
    others = without != 0.0
    for call in (cross_entropy(t, "none"), distillation(logits, tokens, 2.0, "none")):
        def gradients(back):
            a, b = x.clone().requires_grad_(), w.clone().requires_grad_(not frozen)
            return torch.autograd.grad(call(a, b), (a,) if frozen else (a, b), back)
        got, want = gradients(spoilt), gradients(without)
        assert torch.equal(got[0][others], want[0][others]) and want[0].isfinite().all()
        assert not got[0][~others].isfinite().any()
        if not frozen:
            assert not got[1].isfinite().any() and want[1].isfinite().all()


@pytest.mark.parametrize("dtype,least", [(torch.float32, -30), (torch.float32, -12), (torch.float16, -5), (torch.bfloat16, -30)])
def test_a_row_s_gradient_does_not_depend_on_the_weights_of_others(dtype, least):
    """Weights over many powers of ten: each row's gradient loses what it would lose alone."""
    rows = 60
    x, w, t = inputs(rows, 3000, 72, dtype)
    t = t.clamp(min=0)
    dloss = 10.0 ** torch.linspace(least, 0, rows, device="cuda") * torch.where(torch.arange(rows, device="cuda") % 3 == 0, -1.0, 1.0)
    if dtype == torch.float16:
        dloss = dloss * 1024  # (what a loss scaler leaves room for: gradients that the type can hold)
    for targets, logits, call in ((t, None, cross_entropy(t, "none")), (*reversed(teacher(rows, 5, 3000, dtype)), None)):
        if call is None:
            call = distillation(logits, targets, 2.0, "none")
        out = run(call, x, w, dloss)
        each_row_alone(out, x, w, targets, dloss, range(rows), logits, 1.0 if logits is None else 2.0)
        want = plain.losses(x, w, targets, logits, 1.0 if logits is None else 2.0, "none", dloss)
        plain.within(out["dw"], want["dw"], "dw")


@pytest.mark.parametrize("dtype", DTYPES)
def test_weights_at_the_ends_of_their_range(dtype):
    """The largest and the smallest numbers that there are, and a matrix that is frozen or not."""
    x, w, t = inputs(40, 300, 64, dtype)
    t = t.clamp(min=0)
    dloss = torch.full((40,), 1e-44, device="cuda")
    dloss[3], dloss[4] = 1e-38, 0.0
    if dtype != torch.float16:
        dloss[5], dloss[6] = 2.9e38, -1.8e38
        x[5:7], w = x[5:7] * 0.01, w * 0.01
    out = run(cross_entropy(t, "none"), x, w, dloss)
    assert out["dx"].isfinite().all() and out["dw"].isfinite().all() and not out["dx"][4].any()
    if dtype != torch.float16:
        each_row_alone(out, x, w, t, dloss, (5, 6))


@pytest.mark.parametrize("dtype", DTYPES)
def test_many_rows_with_weights_of_their_own(dtype):
    """More rows than are looked at at once, the largest weight at their end; only one of the gradients."""
    rows = 9001
    x, w, t = inputs(rows, 300, 72, dtype)
    dloss = 10.0 ** (-4 * torch.rand(rows, device="cuda", generator=gen(5)))
    dloss[-1], t[-1] = 30.0, 7
    out, want = run(cross_entropy(t, "none"), x, w, dloss), plain.losses(x, w, t, reduction="none", dloss=dloss)
    for name in want:
        plain.within(out[name], want[name], name)
    a, b = x.clone().requires_grad_(), w.clone().requires_grad_()
    (dx,) = torch.autograd.grad(ops.linear_cross_entropy(a, w, t, reduction="none"), a, dloss)
    (dw,) = torch.autograd.grad(ops.linear_cross_entropy(x, b, t, reduction="none"), b, dloss)
    assert torch.equal(dx, out["dx"]) and torch.equal(dw, out["dw"])


@pytest.mark.parametrize("dtype", DTYPES)
def test_graphs_of_losses_of_each_row(dtype):
    """Two graphs at once, replayed with other rows, weights and targets than they were captured with, beside eager calls on a third stream."""
    rows, v, h = 150, 2000, 136
    states, streams = [], [torch.cuda.Stream() for _ in range(3)]
    for i, s in enumerate(streams):
        x, w, t = inputs(rows, v, h, dtype, seed=10 * i)
        back = torch.ones(rows, device="cuda")
        torch.cuda.synchronize()
        with torch.cuda.stream(s):
            run(cross_entropy(t, "none"), x, w, back)
        torch.cuda.synchronize()
        graph, out = torch.cuda.CUDAGraph(), None
        if i < 2:
            with torch.cuda.graph(graph, stream=s):
                out = run(cross_entropy(t, "none"), x, w, back)
        states.append((graph, x, w, t, back, out))
    for turn in range(3):
        for i, (_, x, w, t, back, _) in enumerate(states):
            other, _, targets = inputs(rows, v, h, dtype, seed=100 * turn + i)
            x.copy_(other * 10.0 ** turn)
            t.copy_(targets)
            back.copy_(10.0 ** (-3 * turn * torch.rand(rows, device="cuda", generator=gen(turn))))
        want = [run(cross_entropy(t, "none"), x, w, back) for _, x, w, t, back, _ in states]
        torch.cuda.synchronize()
        for s, state in zip(streams[:2], states):
            with torch.cuda.stream(s):
                state[0].replay()
        with torch.cuda.stream(streams[2]):
            third = run(cross_entropy(states[2][3], "none"), *states[2][1:3], states[2][4])
        torch.cuda.synchronize()
        for got, expected in zip((states[0][5], states[1][5], third), want):
            assert all(torch.equal(got[name], expected[name]) for name in expected)


# ---- which way a call takes, and what it may lose there --------------------------------------------------

def loses_its_own_rounding(out, want, dtype, what=""):
    for name in ("dx", "dw"):
        exact = want[name][0]
        rounded = (exact.to(dtype).double() - exact).norm()
        # P in two parts is off by 2^-16 at most, the softmax by what its logits are: with at most 4096 products of about 0.03 that may lose 2^-23 of themselves 256 times, 1e-5, beside roundings of
        # at least 2^-13 in the mean.
        assert (out[name].double() - exact).norm() <= 1.1 * rounded + 1e-30, f"{what} {name}"


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("rows,vocabulary,width", [(1, 152064, 1024), (12, 152064, 1024), (64, 262144, 512)])
def test_gradients_of_few_rows_over_a_large_vocabulary(dtype, rows, vocabulary, width):
    x, w, t = inputs(rows, vocabulary, width, dtype)
    dloss = torch.randn(rows, device="cuda", generator=gen(9))
    out = run(cross_entropy(t, "none"), x, w, dloss)
    loses_its_own_rounding(out, plain.losses(x, w, t, reduction="none", dloss=dloss), dtype)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("rows,vocabulary,width", [(5, 257, 64), (129, 255, 65), (300, 5000, 72), (1000, 700, 1003), (33, 20011, 80), (513, 1025, 392)])
def test_gradients_of_small_products_lose_their_own_rounding_alone(dtype, rows, vocabulary, width):
    x, w, t = inputs(rows, vocabulary, width, dtype)
    logits, tokens = teacher(rows, 4, vocabulary, dtype)
    assert not made_with_the_loss(x, w, t)
    one = torch.ones((), device="cuda")
    for targets, kind, call in ((t, None, cross_entropy(t, "mean")), (tokens, logits, distillation(logits, tokens, 1.0, "sum"))):
        loses_its_own_rounding(run(call, x, w, one), plain.losses(x, w, targets, kind, reduction="mean" if kind is None else "sum", dloss=one), dtype)


def test_gradients_of_few_rows_made_with_the_loss():
    """One loss for all rows, few of them: the exponentials are rounded once, what is divided by their sums is not."""
    rows, v, h = 12, 152064, 1024
    x, w, t = inputs(rows, v, h, torch.bfloat16)
    assert made_with_the_loss(x, w, t)
    one = torch.ones((), device="cuda")
    out, want = run(cross_entropy(t, "mean"), x, w, one), plain.losses(x, w, t, dloss=one)
    for name in ("loss", "dx", "dw"):
        plain.within(out[name], want[name], name)
    a, c = x.double(), (t >= 0).double()[:, None] / int((t >= 0).sum())
    q = torch.softmax(a @ w.double().t(), -1).scatter(1, t.clamp(min=0)[:, None], 0.0) * c
    for name, p, m in (("dx", q, w), ("dw", q.t(), a)):
        exact = want[name][0]
        rounded = (exact.bfloat16().double() - exact).norm()
        # Each other word's exponential is off by half a step, 2^-8, and its row's factor by as much; as independent numbers, of which the norm is the root of the sum of squares.
        spread = ((p ** 2) @ (m.double() ** 2)).sum().sqrt()
        assert (out[name].double() - exact).norm() <= 1.1 * rounded + 2.1 * 2.0 ** -8 * spread + 2.0 ** -8 * (p @ m.double()).norm(), name


# ---- waits of gradients made with the loss ---------------------------------------------------------------

def both(x, w, t, wait_ns):
    """The C interface: the mean loss with its gradients, with waits of `wait_ns`."""
    lib, rows = nn.load(), x.shape[0]
    loss, dx, dw = torch.zeros((), device="cuda"), torch.zeros_like(x), torch.zeros_like(w)
    c = VocabularyLoss(dtype=2, x=x.data_ptr(), x_stride=x.stride(0), weight=w.data_ptr(), weight_stride=w.stride(0), tokens=rows, width=x.shape[1], vocabulary=w.shape[0], targets=t.data_ptr(),
                       target_bytes=8, target_strides=(LL * 2)(1, 1), temperature=1.0, reduction=1, loss=loss.data_ptr(), x_grad=dx.data_ptr(), weight_grad=dw.data_ptr())
    floats, size = ctypes.c_size_t(), ctypes.c_size_t()
    assert lib.b2_vocabulary_loss_sizes(ctypes.byref(c), 0, ctypes.byref(floats), None) == 0
    assert lib.b2_vocabulary_loss_both_workspace(ctypes.byref(c), ctypes.byref(size)) == 0 and size.value != 0
    kept, workspace = torch.zeros(floats.value, device="cuda"), torch.zeros(size.value, dtype=torch.uint8, device="cuda")
    c.kept, c.workspace = kept.data_ptr(), workspace.data_ptr()
    assert lib.b2_vocabulary_loss_within(ctypes.byref(c), 2, ctypes.c_ulonglong(wait_ns), ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)) == 0
    torch.cuda.synchronize()
    return {"loss": loss, "dx": dx, "dw": dw}


def test_a_wait_of_gradients_made_with_the_loss_that_runs_out():
    """Without any time a wait may be over or not when it is looked at. Results are right or NaN; where the logits were not done in time they are made again, and may be right then; the status says that a wait
    ran out whenever anything is NaN."""
    x, w, t = inputs(4096, 1024, 32768, torch.bfloat16)
    ops.check_async_error()
    want = plain.losses(x, w, t, dloss=torch.ones((), device="cuda"))
    for name, value in both(x, w, t, 2 * 10 ** 9).items():
        plain.within(value, want[name], name)
    ops.check_async_error()
    ran_out = 0
    for _ in range(40):
        got = both(x, w, t, 0)
        nan = False
        for name, (value, bound) in want.items():
            there = ~got[name].isnan()
            assert ((got[name].double() - value).abs() <= bound)[there].all(), name
            nan |= not bool(there.all())
        try:
            ops.check_async_error()
            assert not nan
        except nn.B200CclError as e:
            assert "ran out" in str(e)
            ran_out += 1
    assert ran_out > 0
    for name, value in both(x, w, t, 2 * 10 ** 9).items():
        plain.within(value, want[name], name)
    ops.check_async_error()


# ---- memory ----------------------------------------------------------------------------------------------

def test_a_loss_that_makes_no_gradients_allocates_none():
    """A small product's gradients are made in the backward pass: nothing of their size is asked for before."""
    x, w, t = inputs(16, 30000, 1024, torch.bfloat16)
    assert not made_with_the_loss(x, w, t)
    x, w = x.requires_grad_(), w.requires_grad_()
    ops.linear_cross_entropy(x, w, t)
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    loss = ops.linear_cross_entropy(x, w, t)
    assert torch.cuda.max_memory_allocated() - before < w.numel() * 2 / 4
    assert loss.isfinite()


def test_exponentials_of_a_vocabulary_that_is_too_large_are_not_kept():
    """256 rows of them would be 1.5 GB: such a loss makes its gradients by pieces of the vocabulary."""
    rows, v, h = 256, 3_000_000, 16
    w, x = normal((v, h), torch.bfloat16, 1, 0.5), normal((rows, h), torch.bfloat16, 2)
    t = torch.randint(0, v, (rows,), device="cuda", generator=gen(3))
    assert made_with_the_loss(x[:64], w, t[:64])
    x, w = x.requires_grad_(), w.requires_grad_()
    torch.cuda.synchronize()
    torch.cuda.empty_cache()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    loss = ops.linear_cross_entropy(x, w, t)
    dx, dw = torch.autograd.grad(loss, (x, w))
    assert torch.cuda.max_memory_allocated() - before < 1 << 30
    want, exact = 0.0, torch.zeros(rows, h, dtype=torch.float64, device="cuda")
    off = torch.zeros_like(exact)
    m = w.detach().double()
    for at in range(0, rows, 32):
        z = x.detach()[at:at + 32].double() @ m.t()
        lse = torch.logsumexp(z, -1, keepdim=True)
        want += float((lse - z.gather(1, t[at:at + 32, None])).sum()) / rows
        p = torch.exp(z - lse).scatter_add_(1, t[at:at + 32, None], -torch.ones(32, 1, dtype=torch.float64, device="cuda")) / rows
        exact[at:at + 32] = p @ m
        off[at:at + 32] = p.abs() @ m.abs()
    assert abs(float(loss.detach()) - want) <= 2.0 ** -18 * want
    # P's rounding, the result's, and what 32-bit sums of three million words lose.
    assert ((dx.double() - exact).abs() <= 2.0 ** -8 * exact.abs() + (2.0 ** -8 + 2.0 ** -9) * off).all()
    assert dw.isfinite().all()


# ---- the model, large enough for gradients that are made with the loss -----------------------------------

def large_model():
    torch.manual_seed(0)
    model = TinyGPT2(vocab=50257, context=40, hidden=768, layers=1, heads=12, vocabulary="fused").cuda()
    with torch.no_grad():
        model.wte.weight.mul_(0.05)
    g = torch.Generator().manual_seed(1)
    tokens, targets = (torch.randint(0, 50257, (3, 40), generator=g).cuda() for _ in range(2))
    targets[0, 30:] = -1
    return model, tokens, targets


def counted(calls):
    prototype = ctypes.CFUNCTYPE(ctypes.c_int, ctypes.c_void_p, ctypes.c_void_p)
    return replaced("b2_vocabulary_loss_both", prototype, lambda original, *arguments: calls.append(1) or original(*arguments))


def test_a_large_model_under_autocast():
    model, tokens, targets = large_model()
    seen, calls = [], []

    def keep(module, arguments, output):
        output.retain_grad()
        seen.append(output)

    model.ln_f.register_forward_hook(keep)
    with counted(calls):
        with torch.autocast("cuda", dtype=torch.bfloat16):
            loss = model(tokens, targets)
        loss.backward()
    assert len(calls) == 1
    x, w, one = seen[0].detach().bfloat16().view(120, 768), model.wte.weight.detach().bfloat16(), torch.ones((), device="cuda")
    want = plain.losses(x, w, targets.view(-1), dloss=one)
    plain.within(loss, want["loss"], "loss")
    plain.within(seen[0].grad.bfloat16().view(120, 768), want["dx"], "dx")  # (a 16-bit gradient, cast to 32 bits)
    untouched = torch.ones(50257, dtype=torch.bool, device="cuda")
    untouched[tokens.view(-1)] = False  # rows of the tied matrix that were not looked up: the loss's gradient alone
    value, bound = want["dw"]
    plain.within(model.wte.weight.grad[untouched].bfloat16(), (value[untouched], bound[untouched]), "dw")
    assert all(p.grad.isfinite().all() for p in model.parameters())


def test_a_large_model_under_the_data_parallel_wrapper():
    torch.cuda.set_device(0)
    comm = nn.Communicator(devices=[0], wait_timeout_ms=2000)
    model, tokens, targets = large_model()
    alone, calls = copy.deepcopy(model), []
    with counted(calls), torch.autocast("cuda", dtype=torch.bfloat16):
        alone(tokens, targets).backward()
        ddp = DistributedDataParallel(model, CclBackend(comm))
        ddp.zero_grad()
        ddp(tokens, targets).backward()
        ddp.finish()
    torch.cuda.synchronize()
    assert len(calls) == 2
    for p, q in zip(model.parameters(), alone.parameters()):
        assert torch.equal(p.grad, q.grad)
    comm.close()
