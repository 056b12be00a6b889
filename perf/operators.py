"""What the speed of the training operators is measured on: activations kept in 8 bits for the backward pass (the
codec, GELU, the weight gradient of a projection) and the position rotation of queries and keys, alone and with their norms.

A case is a plain dict. All have

  op      checkpoint | gelu | weight_grad | rotary | qk_norm
  dtype   float | fp16 | bf16, of every floating input and output
  tokens  rows of the activation; of rotary and qk_norm: tokens of each of ``batch`` sequences

and, by operator,

  checkpoint   columns: an activation is packed into 8 bits and read back
  gelu         columns, tanh: forward and backward, the input kept in 8 bits
  weight_grad  inputs, outputs: the input of a projection is packed, then its weight's and bias's gradients are made from it
  rotary       batch, heads, kv_heads, dim, rotated, interleaved, offset (first position), scaled (frequencies and
               magnitude stretched for long contexts), train (also the gradients of queries and keys)
  qk_norm      the same, with the norm of each head before the rotation; train: the inputs are kept in 8 bits, and the weights' gradients are made too

The 8-bit form of a block of neighbouring elements (32 of a row; of queries and keys: a head) with largest magnitude
``2^a <= amax < 2^(a+1)`` is a power of two ``2^q``, ``q = max(a - 6, -126)`` (-24 for fp16), and whole numbers of at most 127:
``x ~ sign * min(round(|x| / 2^q), 127) * 2^q``, ties to even.
"""
import math

import torch

own = False

DTYPES = {"float": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
BYTES = {"float": 4, "fp16": 2, "bf16": 2}
KEPT = 1 + 1 / 32  # bytes of an element in 8 bits, its share of the block's scale included
EPS = 1e-6


def _rows(name, op, dtype, tokens, **more):
    c = {"op": op, "dtype": dtype, "tokens": tokens, **more}
    return {"name": name, **c} if name else c


def _heads(name, op, dtype, batch, tokens, heads, kv_heads, dim, rotated, interleaved=False, offset=0, scaled=False, train=False):
    return _rows(name, op, dtype, tokens, batch=batch, heads=heads, kv_heads=kv_heads, dim=dim, rotated=rotated,
                 interleaved=interleaved, offset=offset, scaled=scaled, train=train)


def listed():
    return [
        # The hidden state of a short sequence at GPT-2-small's width: the calls themselves.
        _rows("checkpoint_64x768", "checkpoint", "bf16", 64, columns=768),
        # One wide layer's activation of a full batch, kept and read back.
        _rows("checkpoint_16384x4096", "checkpoint", "bf16", 16384, columns=4096),
        # Lengths that are no multiple of anything, in the other 16-bit type and with the other formula.
        _rows("gelu_odd", "gelu", "fp16", 1237, columns=1003, tanh=True),
        # The MLP's activation of a full batch, forward and backward.
        _rows("gelu_8192x8192", "gelu", "bf16", 8192, columns=8192, tanh=False),
        # The attention output projection of GPT-2-small on one short sequence: few output tiles, the token axis is the long one.
        _rows("weight_grad_1024_768", "weight_grad", "bf16", 1024, inputs=768, outputs=768),
        # The joint projection of queries, keys and values of GPT-2-small on eight full contexts, in full precision.
        _rows("weight_grad_8192_768_2304", "weight_grad", "float", 8192, inputs=768, outputs=2304),
        # A wide projection on a full batch: the largest product.
        _rows("weight_grad_16384_4096", "weight_grad", "bf16", 16384, inputs=4096, outputs=4096),
        # One token of one sequence at GPT-2-small's heads, far into a stretched context: latency.
        _heads("rotary_one_token", "rotary", "bf16", 1, 1, 12, 12, 64, 64, offset=100000, scaled=True),
        # A long sequence with shared key heads, forward and backward.
        _heads("rotary_32768", "rotary", "bf16", 1, 32768, 32, 8, 128, 128, scaled=True, train=True),
        # Odd lengths, part of each head, neighbouring pairs, no gradient.
        _heads("qk_norm_odd", "qk_norm", "fp16", 3, 333, 7, 1, 80, 40, interleaved=True, offset=17),
        # Attention inputs of GPT-2-small on eight full contexts, a training step.
        _heads("qk_norm_8x1024", "qk_norm", "bf16", 8, 1024, 12, 12, 64, 64, train=True),
        # The same of a wide layer with shared key heads.
        _heads("qk_norm_4x4096", "qk_norm", "bf16", 4, 4096, 32, 8, 128, 128, train=True),
    ]


def _spread(rng, low, high):
    n = int(math.exp(rng.uniform(math.log(low), math.log(high + 0.999))))
    if n >= 64 and rng.random() < 0.5:
        n = n // 64 * 64
    return max(low, min(high, n))


def draw(rng):
    """One token to 16384 (rotations: 32768), widths of 1 to 8192 (projections: 8 to 4096), heads of 2 to 256 elements, every type; half of the sizes ragged."""
    op = rng.choice(["checkpoint", "gelu", "weight_grad", "weight_grad", "rotary", "qk_norm", "qk_norm"])
    dtype = rng.choice(["float", "fp16", "bf16", "bf16"])
    if op in ("checkpoint", "gelu"):
        columns = _spread(rng, 1, 8192)
        tokens = _spread(rng, 1, min(16384, (1 << 25) // columns))
        return _rows("", op, dtype, tokens, columns=columns, **({"tanh": rng.random() < 0.5} if op == "gelu" else {}))
    if op == "weight_grad":
        inputs, outputs = _spread(rng, 8, 4096), _spread(rng, 8, 4096)
        tokens = _spread(rng, 1, min(16384, (1 << 36) // (inputs * outputs)))
        return _rows("", op, dtype, tokens, inputs=inputs, outputs=outputs)
    dim = rng.choice([32, 48, 64, 64, 80, 96, 128, 128, 128, 256, 2 * rng.randint(1, 128)])
    rotated = dim if rng.random() < 0.6 else 2 * rng.randint(1, dim // 2)
    kv_heads = rng.choice([1, 1, 2, 3, 4, 8])
    heads = kv_heads * rng.choice([1, 1, 2, 4, 7])
    batch = rng.choice([1, 1, 2, 3, 8])
    tokens = _spread(rng, 1, min(32768, (1 << 26) // (batch * (heads + kv_heads) * dim)))
    return _heads("", op, dtype, batch, tokens, heads, kv_heads, dim, rotated, interleaved=rng.random() < 0.5,
                  offset=rng.choice([0, 0, rng.randint(1, 1000000)]), scaled=rng.random() < 0.5, train=rng.random() < 0.6)


class State:
    """The tensors that a training program has in hand, by name."""

    def __init__(self, case, **tensors):
        self.case = case
        self.__dict__.update(tensors)


def _activation(gen, rows, columns, dtype):
    """Normal values under a scale of each column's own, a few of them large, as hidden states have them."""
    x = torch.randn(rows, columns, device="cuda", generator=gen)
    x *= torch.exp(torch.randn(columns, device="cuda", generator=gen))
    return x.clamp_(-1000.0, 1000.0).to(dtype)


def _frequencies(case):
    """Radians per position of each pair, in 64 bits. Scaled: slow pairs are slowed further, by up to 8, between two and sixteen turns in 4096 positions."""
    pairs = case["rotated"] // 2
    f = 10000.0 ** (-torch.arange(pairs, dtype=torch.float64, device="cuda") / pairs)
    if case["scaled"]:
        turns = f * 4096 / (2 * math.pi)
        keep = ((turns - 2.0) / 14.0).clamp(0.0, 1.0)
        f = f * (keep + (1.0 - keep) / 8.0)
    return f


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype = DTYPES[case["dtype"]]
    if case["op"] == "checkpoint":
        return State(case, x=_activation(gen, case["tokens"], case["columns"], dtype))
    if case["op"] == "gelu":
        x = _activation(gen, case["tokens"], case["columns"], dtype).requires_grad_()
        return State(case, x=x, dy=(0.1 * torch.randn(case["tokens"], case["columns"], device="cuda", generator=gen)).to(dtype))
    if case["op"] == "weight_grad":
        return State(case, x=_activation(gen, case["tokens"], case["inputs"], dtype),
                     dy=(0.01 * torch.randn(case["tokens"], case["outputs"], device="cuda", generator=gen)).to(dtype))
    b, t, h, g, d = (case[k] for k in ("batch", "tokens", "heads", "kv_heads", "dim"))
    # Queries and keys lie in the output of one projection, beside the values.
    qkv = torch.randn(b, t, (h + 2 * g) * d, device="cuda", generator=gen).to(dtype)
    q = qkv[..., :h * d].view(b, t, h, d).detach().requires_grad_(case["train"])
    k = qkv[..., h * d:(h + g) * d].view(b, t, g, d).detach().requires_grad_(case["train"])
    s = State(case, q=q, k=k, positions=torch.arange(t, device="cuda") + case["offset"], frequencies=_frequencies(case),
              magnitude=1.0 + 0.1 * math.log(8.0) if case["scaled"] else 1.0, layout="interleaved" if case["interleaved"] else "half")
    if case["train"]:
        s.dq = torch.randn(b, t, h, d, device="cuda", generator=gen).to(dtype)
        s.dk = torch.randn(b, t, g, d, device="cuda", generator=gen).to(dtype)
    if case["op"] == "qk_norm":
        s.wq, s.wk = ((1.0 + 0.1 * torch.randn(d, device="cuda", generator=gen)).to(dtype).requires_grad_(case["train"]) for _ in range(2))
    return s


# -- plain forms: 32 bits, one rounding at the end ---------------------------------------------------------


def _kept(x, block, low):
    """`x` (32 bits) as the values that its 8-bit form stands for."""
    columns = x.shape[-1]
    b = torch.nn.functional.pad(x, (0, -columns % block)).unflatten(-1, (-1, block))
    amax = b.abs().amax(-1, keepdim=True)
    a = (amax.view(torch.int32) >> 23) - 127
    step = ((a - 6).clamp(min=low) + 127 << 23).view(torch.float32)
    m = (b / step).round().clamp(-127.0, 127.0)
    return (m * step).flatten(-2)[..., :columns]


def _low(dtype):
    return -24 if dtype == torch.float16 else -126


def _rotate(x, cos, sin, s):
    """Pairs of the first elements of each head turned by their angles."""
    rotated = 2 * cos.shape[-1]
    head, rest = x[..., :rotated], x[..., rotated:]
    if s.layout == "interleaved":
        u, v = head[..., 0::2], head[..., 1::2]
        turned = torch.stack((u * cos - v * sin, u * sin + v * cos), -1).flatten(-2)
    else:
        u, v = head.chunk(2, -1)
        turned = torch.cat((u * cos - v * sin, u * sin + v * cos), -1)
    return torch.cat((turned, rest), -1)


def _angles(s):
    angle = s.positions.double()[:, None, None] * s.frequencies
    return (s.magnitude * angle.cos()).float(), (s.magnitude * angle.sin()).float()


def _plain(s):
    c = s.case
    dtype = DTYPES[c["dtype"]]
    if c["op"] == "checkpoint":
        return _kept(s.x.float(), 32, _low(dtype)).to(dtype)
    if c["op"] == "gelu":
        x = s.x.float()
        v = _kept(x, 32, _low(dtype))
        if c["tanh"]:
            r = math.sqrt(2.0 / math.pi)
            y = 0.5 * x * (1.0 + torch.tanh(r * (x + 0.044715 * x * x * x)))
            th = torch.tanh(r * (v + 0.044715 * v * v * v))
            slope = 0.5 * (1.0 + th) + 0.5 * v * (1.0 - th * th) * r * (1.0 + 3 * 0.044715 * v * v)
        else:
            y = 0.5 * x * torch.erfc(-x * math.sqrt(0.5))
            slope = 0.5 * torch.erfc(-v * math.sqrt(0.5)) + v * torch.exp(-0.5 * v * v) / math.sqrt(2.0 * math.pi)
        return {"y": y.to(dtype), "dx": (s.dy.float() * slope).to(dtype)}
    if c["op"] == "weight_grad":
        dy = s.dy.float()
        return {"dw": (dy.t() @ _kept(s.x.float(), 32, _low(dtype))).to(dtype), "db": dy.sum(0).to(dtype)}
    cos, sin = _angles(s)
    out = {}
    for name in ("q", "k"):
        x = getattr(s, name).float()
        if c["op"] == "rotary":
            out[name] = _rotate(x, cos, sin, s).to(dtype)
            if c["train"]:
                out["d" + name] = _rotate(getattr(s, "d" + name).float(), cos, -sin, s).to(dtype)
            continue
        w = getattr(s, "w" + name).float()
        out[name] = _rotate(x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * w, cos, sin, s).to(dtype)
        if c["train"]:
            v = _kept(x, c["dim"], _low(dtype))
            rstd = torch.rsqrt(v.square().mean(-1, keepdim=True) + EPS)
            g = _rotate(getattr(s, "d" + name).float(), cos, -sin, s)
            n = v * rstd
            out["dw" + name] = (g * n).sum((0, 1, 2)).to(dtype)
            gw = g * w
            out["d" + name] = (rstd * (gw - n * (gw * n).mean(-1, keepdim=True))).to(dtype)
    return {k: v.detach() for k, v in out.items()}


def run(s):
    c = s.case
    if not own:
        with torch.no_grad():
            return _plain(s)
    from nano_nccl_b200 import ops
    if c["op"] == "checkpoint":
        return ops.unpack8(ops.pack8(s.x))
    if c["op"] == "gelu":
        y = ops.gelu8(s.x, approximate="tanh" if c["tanh"] else "none")
        (dx,) = torch.autograd.grad(y, s.x, s.dy)
        return {"y": y.detach(), "dx": dx}
    if c["op"] == "weight_grad":
        dw, db = ops.weight_grad8(s.dy, ops.pack8(s.x), bias=True)
        return {"dw": dw, "db": db}
    if c["op"] == "rotary":
        q, k = ops.rotary(s.q, s.k, s.positions, s.frequencies, layout=s.layout, magnitude=s.magnitude)
        if not c["train"]:
            return {"q": q, "k": k}
        dq, dk = torch.autograd.grad((q, k), (s.q, s.k), (s.dq, s.dk))
        return {"q": q.detach(), "k": k.detach(), "dq": dq, "dk": dk}
    q, k = ops.qk_norm_rotary(s.q, s.k, s.wq, s.wk, s.positions, s.frequencies, layout=s.layout, magnitude=s.magnitude,
                              eps=EPS, keep="int8" if c["train"] else None)
    if not c["train"]:
        return {"q": q, "k": k}
    dq, dk, dwq, dwk = torch.autograd.grad((q, k), (s.q, s.k, s.wq, s.wk), (s.dq, s.dk))
    return {"q": q.detach(), "k": k.detach(), "dq": dq, "dk": dk, "dwq": dwq, "dwk": dwk}


def work(case):
    e = BYTES[case["dtype"]]
    t = case["tokens"]
    if case["op"] == "checkpoint":  # read, keep; read what was kept, write
        return {"bytes": 2 * t * case["columns"] * (e + KEPT), "flops": 4 * t * case["columns"]}
    if case["op"] == "gelu":  # x -> y and what is kept; dy and what was kept -> dx
        return {"bytes": t * case["columns"] * (4 * e + 2 * KEPT), "flops": 30 * t * case["columns"]}
    if case["op"] == "weight_grad":  # x -> what is kept; dy and what was kept -> dw, db
        i, o = case["inputs"], case["outputs"]
        return {"bytes": t * i * (e + 2 * KEPT) + t * o * e + (i + 1) * o * e, "flops": 2 * t * i * o}
    rows = case["batch"] * t * (case["heads"] + case["kv_heads"])
    n = rows * case["dim"]
    b = 2 * n * e + 8 * t + 4 * case["rotated"]
    f = 3 * rows * case["rotated"]
    if case["op"] == "qk_norm":
        b += 2 * case["dim"] * e
        f += 4 * n
    if case["train"]:
        b += 2 * n * e
        f += 3 * rows * case["rotated"]
        if case["op"] == "qk_norm":
            b += 2 * n * (1 + 1 / case["dim"]) + 4 * case["dim"] * e
            f += 12 * n
    return {"bytes": b, "flops": f}


# -- the definitions in 64 bits ----------------------------------------------------------------------------


def _exact_kept(x, block, dtype):
    """Block by block: the exponent from frexp, the quotient and its rounding in 64 bits."""
    lead, columns = x.shape[:-1], x.shape[-1]
    blocks = -(-columns // block)
    b = torch.zeros(*lead, blocks * block, dtype=torch.float64, device=x.device)
    b[..., :columns] = x
    b = b.view(*lead, blocks, block)
    _, e = torch.frexp(b.abs().max(-1, keepdim=True).values)  # amax in [2^(e-1), 2^e)
    q = torch.clamp(e.to(torch.int64) - 7, min=-24 if dtype == torch.float16 else -126)
    step = ((q + 1023) << 52).view(torch.float64)  # (a power function is a rounding off, which decides ties)
    return (torch.sign(b) * torch.minimum(torch.round(b.abs() / step), torch.full_like(b, 127.0)) * step).view(*lead, -1)[..., :columns]


def _exact_turn(x, s):
    """Every pair as a complex number, times magnitude * exp(i angle)."""
    n = s.frequencies.numel()
    angle = s.positions.to(torch.float64).view(1, -1, 1, 1) * s.frequencies
    turn = torch.polar(torch.full_like(angle, s.magnitude), angle)
    if s.layout == "interleaved":
        z = torch.view_as_complex(x[..., :2 * n].reshape(*x.shape[:-1], n, 2).contiguous()) * turn
        first = torch.view_as_real(z).reshape(*x.shape[:-1], 2 * n)
    else:
        z = torch.complex(x[..., :n].contiguous(), x[..., n:2 * n].contiguous()) * turn
        first = torch.cat([z.real, z.imag], dim=-1)
    return torch.cat([first, x[..., 2 * n:]], dim=-1)


def exact(case, seed):
    s = prepare(case, seed)
    dtype = DTYPES[case["dtype"]]
    if case["op"] == "checkpoint":
        return _exact_kept(s.x.double(), 32, dtype)
    if case["op"] == "gelu":
        def gelu(v):
            if case["tanh"]:
                return v * torch.sigmoid(2.0 * math.sqrt(2.0 / math.pi) * (v + 0.044715 * v.pow(3)))
            return v * torch.special.ndtr(v)
        x = s.x.detach().double()
        v = _exact_kept(x, 32, dtype).requires_grad_()
        (dx,) = torch.autograd.grad(gelu(v), v, s.dy.double())
        return {"y": gelu(x), "dx": dx}
    if case["op"] == "weight_grad":
        dy = s.dy.double()
        return {"dw": torch.mm(dy.t(), _exact_kept(s.x.double(), 32, dtype)), "db": torch.mv(dy.t(), torch.ones_like(dy[:, 0]))}
    out = {}
    for name in ("q", "k"):
        x = getattr(s, name).detach().double()

        def forward(v, w):
            if w is not None:
                v = v / torch.sqrt((v * v).sum(-1, keepdim=True) / case["dim"] + EPS) * w
            return _exact_turn(v, s)

        w = getattr(s, "w" + name).detach().double() if case["op"] == "qk_norm" else None
        out[name] = forward(x, w)
        if case["train"]:
            dy = getattr(s, "d" + name).double()
            if w is None:
                v = x.requires_grad_()
                (out["d" + name],) = torch.autograd.grad(forward(v, None), v, dy)
            else:
                v, w = _exact_kept(x, case["dim"], dtype).requires_grad_(), w.requires_grad_()
                out["d" + name], out["dw" + name] = torch.autograd.grad(forward(v, w), (v, w), dy)
    return {k: v.detach() for k, v in out.items()}
