"""What the speed of the operators at the two ends of a training step is measured on: the lookup of tokens in an embedding with its
gradient, and the two losses over a vocabulary that never store the logits, cross entropy and distillation from a teacher's top logits.

A case is a plain dict. All have

  op          embedding | cross_entropy | distillation
  dtype       float | fp16 | bf16, of every floating input and output but the loss, which is float
  tokens      rows
  vocabulary, width   of the matrix that tokens are looked up in, or that makes logits of hidden states
  padded      the share of rows that stand for no token (-1): a batch of sequences of several lengths
  train       also the gradients

and, by operator,

  embedding      scale
  cross_entropy  reduction: mean (over rows with a target) | none (a loss for each row)
  distillation   the same, entries (of the teacher, for each row) and temperature

Cross entropy of a row is ``log sum exp(z) - z[target]`` with ``z = x @ weight.T``. Distillation is ``temperature^2`` times the divergence
``sum p (log p - log q)``, p being the softmax of the row's teacher logits / temperature over its entries and q that of z / temperature over the vocabulary.
"""
import math

import torch

own = False

DTYPES = {"float": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
BYTES = {"float": 4, "fp16": 2, "bf16": 2}


def _case(name, op, dtype, tokens, vocabulary, width, padded=0.0, train=True, **more):
    c = {"op": op, "dtype": dtype, "tokens": tokens, "vocabulary": vocabulary, "width": width, "padded": padded, "train": train, **more}
    return {"name": name, **c} if name else c


def listed():
    return [
        # The token that was chosen last goes back in, GPT-2-small: the call itself.
        _case("embedding_one_token", "embedding", "bf16", 1, 50257, 768, train=False, scale=1.0),
        # Lengths that are no multiple of anything, a width whose rows start at odd addresses, padded sequences.
        _case("embedding_odd", "embedding", "fp16", 3 * 333, 32003, 1003, padded=0.2, scale=math.sqrt(1003.0)),
        # GPT-2-small, a training step of eight full contexts.
        _case("embedding_8x1024", "embedding", "bf16", 8192, 50257, 768, scale=1.0),
        # A wide model with a large vocabulary, a training step.
        _case("embedding_32768_wide", "embedding", "bf16", 32768, 131072, 4096, scale=64.0),
        # The smallest model that this repository trains, on two of its contexts, in full precision.
        _case("cross_entropy_tiny", "cross_entropy", "float", 2 * 64, 512, 64, reduction="mean"),
        # GPT-2-small's loss on one context while it is evaluated: each token's own, no gradient.
        _case("cross_entropy_eval_1024", "cross_entropy", "bf16", 1024, 50257, 768, train=False, reduction="none"),
        # Ragged everything, and rows that are weighted one by one.
        _case("cross_entropy_odd", "cross_entropy", "fp16", 777, 32003, 1003, padded=0.1, reduction="none"),
        # GPT-2-small, a training step of eight contexts, some of them padded.
        _case("cross_entropy_8x1024", "cross_entropy", "bf16", 8192, 50257, 768, padded=0.05, reduction="mean"),
        # The same model in full precision, on two contexts.
        _case("cross_entropy_2x1024_float", "cross_entropy", "float", 2048, 50257, 768, reduction="mean"),
        # A wide model with a large vocabulary: the largest products.
        _case("cross_entropy_4096_wide", "cross_entropy", "bf16", 4096, 131072, 4096, reduction="mean"),
        # A small student, few entries, some of them missing.
        _case("distillation_odd", "distillation", "fp16", 333, 1009, 80, padded=0.1, entries=7, temperature=1.5, reduction="none"),
        # GPT-2-small as the student of a teacher whose 32 largest logits were stored.
        _case("distillation_8x1024", "distillation", "bf16", 8192, 50257, 768, entries=32, temperature=2.0, reduction="mean"),
    ]


def _spread(rng, low, high):
    n = int(math.exp(rng.uniform(math.log(low), math.log(high + 0.999))))
    if n >= 64 and rng.random() < 0.5:
        n = n // 64 * 64
    return max(low, min(high, n))


def draw(rng):
    """One row to 32768 (losses: 16384), vocabularies of 2 to 131072, widths of 8 to 4096, every type; half of the sizes ragged."""
    op = rng.choice(["embedding", "embedding", "cross_entropy", "cross_entropy", "distillation"])
    dtype = rng.choice(["float", "fp16", "bf16", "bf16"])
    padded = rng.choice([0.0, 0.0, 0.1, 0.5])
    train = rng.random() < 0.8
    vocabulary, width = _spread(rng, 2, 131072), _spread(rng, 8, 4096)
    if op == "embedding":
        tokens = _spread(rng, 1, min(32768, (1 << 27) // width))
        return _case("", op, dtype, tokens, vocabulary, width, padded, train, scale=rng.choice([1.0, 1.0, math.sqrt(width)]))
    # float takes six times the products.
    most = (1 << 41) // (16 if dtype == "float" else 1)
    tokens = _spread(rng, 1, max(1, min(16384, (1 << 29) // vocabulary, most // (vocabulary * width))))
    more = {"reduction": rng.choice(["mean", "mean", "none"])}
    if op == "distillation":
        more.update(entries=_spread(rng, 1, min(128, vocabulary)), temperature=rng.choice([1.0, 1.0, 2.0, 3.5]))
    return _case("", op, dtype, tokens, vocabulary, width, padded, train, **more)


class State:
    """The tensors that a training program has in hand, by name."""

    def __init__(self, case, **tensors):
        self.case = case
        self.__dict__.update(tensors)


def _tokens(gen, case, count):
    """Tokens as text has them: the n-th most frequent about n times as rare as the first, in no order of their numbers."""
    v = case["vocabulary"]
    rank = torch.exp(torch.rand(count, device="cuda", generator=gen, dtype=torch.float64) * math.log(v + 1.0)).long().sub_(1).clamp_(0, v - 1)
    step = next(s for s in (7919, 104729, 1299709, 1) if s == 1 or math.gcd(s, v) == 1)
    tokens = rank * step % v
    if case["padded"] > 0.0:  # the ends of sequences
        absent = torch.rand(count, device="cuda", generator=gen) < case["padded"]
        tokens = torch.where(absent, torch.full_like(tokens, -1), tokens)
    return tokens


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype = DTYPES[case["dtype"]]
    t, v, h = case["tokens"], case["vocabulary"], case["width"]
    tokens = _tokens(gen, case, t)
    # Logits of hidden states of norm sqrt(width) have a standard deviation of two.
    weight = (2.0 / math.sqrt(h) * torch.randn(v, h, device="cuda", generator=gen)).to(dtype)
    s = State(case, weight=weight.requires_grad_(case["train"]))
    if case["op"] == "embedding":
        s.tokens = tokens
        if case["train"]:
            s.dy = (0.01 * torch.randn(t, h, device="cuda", generator=gen)).to(dtype)
        return s
    # Hidden states that know something of their targets: some rows much, some little.
    known = torch.rand(t, 1, device="cuda", generator=gen) * 2.5
    x = torch.randn(t, h, device="cuda", generator=gen) + known * weight.detach()[tokens.clamp(min=0)].float()
    s.x = x.to(dtype).requires_grad_(case["train"])
    if case["op"] == "cross_entropy":
        s.targets = tokens
    else:
        k = case["entries"]
        # k tokens of the vocabulary, the target first; the teacher is sure of some rows and not of others.
        step = torch.randint(1, max(2, v // k + 1), (t, 1), device="cuda", generator=gen)
        s.teacher_tokens = (tokens.clamp(min=0)[:, None] + torch.arange(k, device="cuda") * step) % v
        absent = (tokens < 0)[:, None] | (torch.rand(t, k, device="cuda", generator=gen) < 0.2 * (case["padded"] > 0.0))
        s.teacher_tokens = torch.where(absent, torch.full_like(s.teacher_tokens, -1), s.teacher_tokens)
        spread = 1.0 + 4.0 * torch.rand(t, 1, device="cuda", generator=gen)
        s.teacher_logits = (10.0 + spread * torch.randn(t, k, device="cuda", generator=gen).sort(-1, descending=True).values).to(dtype)
    if case["train"]:
        # What comes back to the loss: 1, or a weight for each row.
        s.dloss = torch.rand(t, device="cuda", generator=gen) / t if case["reduction"] == "none" else torch.ones((), device="cuda")
    return s


# -- plain forms: 32 bits, one rounding at the end ---------------------------------------------------------


def _plain(s):
    c = s.case
    dtype = DTYPES[c["dtype"]]
    w = s.weight.float()
    if c["op"] == "embedding":
        there = (s.tokens >= 0).float()[:, None]
        index = s.tokens.clamp(min=0)
        out = {"y": (c["scale"] * w[index] * there).to(dtype)}
        if c["train"]:
            out["dw"] = torch.zeros_like(w).index_add_(0, index, c["scale"] * s.dy.float() * there).to(dtype)
        return out
    x = s.x.float()
    tau = c.get("temperature", 1.0)
    z = x @ w.t()
    z /= tau
    top = z.max(-1, keepdim=True).values
    e = torch.exp(z - top)
    total = e.sum(-1, keepdim=True)
    lse = top + torch.log(total)
    if c["op"] == "cross_entropy":
        index, there = s.targets.clamp(min=0)[:, None], (s.targets >= 0)[:, None]
        p = there.float()
        loss = (p * (lse - z.gather(-1, index))).squeeze(-1)
    else:
        index, present = s.teacher_tokens.clamp(min=0), s.teacher_tokens >= 0
        there = present.any(-1, keepdim=True)
        logits = torch.where(present, s.teacher_logits.float() / tau, torch.full_like(s.teacher_logits, -math.inf, dtype=torch.float32))
        logits = logits - torch.where(there, logits.max(-1, keepdim=True).values, torch.zeros_like(lse))
        p = torch.exp(logits)
        sums = p.sum(-1, keepdim=True)
        sums = torch.where(there, sums, torch.ones_like(sums))
        log_p = torch.where(present, logits - torch.log(sums), torch.zeros_like(logits))
        p = p / sums
        loss = tau * tau * (p * (log_p - z.gather(-1, index) + lse)).sum(-1)
    mean = c["reduction"] == "mean"
    count = there.sum().clamp(min=1).float()
    out = {"loss": loss.sum() / count if mean else loss}
    if c["train"]:
        scale = tau * there.float() * (s.dloss / count if mean else s.dloss[:, None])
        dz = e.div_(total)
        dz.scatter_add_(-1, index, -p)
        dz *= scale
        out["dx"] = (dz @ w).to(dtype)
        out["dw"] = (dz.t() @ x).to(dtype)
    return out


def run(s):
    c = s.case
    if not own:
        with torch.no_grad():
            return _plain(s)
    from nano_nccl_b200 import ops
    if c["op"] == "embedding":
        y = ops.embedding(s.tokens, s.weight, scale=c["scale"])
        if not c["train"]:
            return {"y": y}
        (dw,) = torch.autograd.grad(y, s.weight, s.dy)
        return {"y": y.detach(), "dw": dw}
    if c["op"] == "cross_entropy":
        loss = ops.linear_cross_entropy(s.x, s.weight, s.targets, reduction=c["reduction"])
    else:
        loss = ops.linear_distillation(s.x, s.weight, s.teacher_logits, s.teacher_tokens, temperature=c["temperature"], reduction=c["reduction"])
    if not c["train"]:
        return {"loss": loss}
    dx, dw = torch.autograd.grad(loss, (s.x, s.weight), s.dloss)
    return {"loss": loss.detach(), "dx": dx, "dw": dw}


def work(case):
    e = BYTES[case["dtype"]]
    t, v, h = case["tokens"], case["vocabulary"], case["width"]
    if case["op"] == "embedding":  # tokens, their rows -> y; dy -> the whole gradient
        b, f = 8 * t + 2 * t * h * e, t * h
        if case["train"]:
            b += 8 * t + (t + v) * h * e
            f += t * h
        return {"bytes": b, "flops": f}
    b = (t + v) * h * e + (8 * t if case["op"] == "cross_entropy" else t * case["entries"] * (8 + e)) + 4 * t
    f = 2 * t * v * h
    if case["train"]:
        b += (t + v) * h * e + 4 * t
        f *= 3
    return {"bytes": b, "flops": f}


# -- the definitions in 64 bits ----------------------------------------------------------------------------


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "embedding":
        w = s.weight.detach().double()
        inside = torch.nonzero(s.tokens >= 0).squeeze(-1)
        y = torch.zeros(case["tokens"], case["width"], dtype=torch.float64, device="cuda")
        y[inside] = torch.index_select(w, 0, s.tokens[inside]) * case["scale"]
        if not case["train"]:
            return {"y": y}
        # Rows in the order of their tokens, and sums over each token's segment.
        tokens, order = torch.sort(s.tokens[inside], stable=True)
        rows = s.dy[inside][order].double()
        dw = torch.zeros_like(w)
        if tokens.numel():
            unique, lengths = torch.unique_consecutive(tokens, return_counts=True)
            dw[unique] = torch.segment_reduce(rows, "sum", lengths=lengths, axis=0) * case["scale"]
        return {"y": y, "dw": dw}
    train = case["train"]
    w = s.weight.detach().double().requires_grad_(train)
    tau = case.get("temperature", 1.0)
    t, v = case["tokens"], case["vocabulary"]
    losses, dx = [], []
    dw = torch.zeros_like(w) if train else None
    present = s.targets[:, None] >= 0 if case["op"] == "cross_entropy" else s.teacher_tokens >= 0
    counted = present.any(-1)
    count = max(1, int(counted.sum()))
    rows = max(1, (1 << 27) // v)
    for at in range(0, t, rows):
        part = slice(at, min(t, at + rows))
        x = s.x.detach()[part].double().requires_grad_(train)
        log_q = torch.log_softmax(torch.nn.functional.linear(x, w) / tau, dim=-1)
        if case["op"] == "cross_entropy":
            loss = torch.nn.functional.nll_loss(log_q, torch.where(counted[part], s.targets[part], -100), ignore_index=-100, reduction="none")
        else:
            # The teacher's distribution over its own entries; what is absent weighs nothing.
            logits = s.teacher_logits[part].double() / tau
            log_p = torch.log_softmax(logits.masked_fill(~present[part], -1e300), dim=-1).masked_fill(~present[part], 0.0)
            p = log_p.exp().masked_fill(~present[part], 0.0)
            loss = tau ** 2 * (p * (log_p - log_q.gather(1, s.teacher_tokens[part].clamp(min=0)))).sum(-1)
        losses.append(loss.detach())
        if train:
            back = counted[part].double() * (s.dloss.double() / count if case["reduction"] == "mean" else s.dloss[part].double())
            gx, gw = torch.autograd.grad(loss, (x, w), back)
            dx.append(gx)
            dw += gw
    loss = torch.cat(losses)
    out = {"loss": loss.sum() / count if case["reduction"] == "mean" else loss}
    if train:
        out.update(dx=torch.cat(dx), dw=dw.detach())
    return out
