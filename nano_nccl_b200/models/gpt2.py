"""GPT-2-small layer stack: the list of parameter shapes (124M elements: hidden 768, 12 layers,
vocabulary 50257, context 1024) used as the gradient list of the bucketed all-reduce benchmark, and
a tiny trainable module of the same structure for data-parallel smoke tests."""
import torch

from .. import ops


def gpt2_small_shapes(hidden=768, layers=12, vocab=50257, context=1024):
    shapes = [(vocab, hidden), (context, hidden)]
    for _ in range(layers):
        shapes += [(hidden,), (hidden,),                       # ln_1
                   (hidden, 3 * hidden), (3 * hidden,),        # attn.c_attn
                   (hidden, hidden), (hidden,),                # attn.c_proj
                   (hidden,), (hidden,),                       # ln_2
                   (hidden, 4 * hidden), (4 * hidden,),        # mlp.c_fc
                   (4 * hidden, hidden), (hidden,)]            # mlp.c_proj
    shapes += [(hidden,), (hidden,)]                           # ln_f
    return shapes


class _Linear8(torch.nn.Linear):
    """A projection whose input is kept in 8 bits."""

    def forward(self, x):
        return ops.linear8(x, self.weight, self.bias)


class _Gelu8(torch.nn.GELU):
    """GELU whose input is kept in 8 bits."""

    def forward(self, x):
        return ops.gelu8(x, self.approximate)


class _Embedding(torch.nn.Embedding):
    """Tokens looked up by :func:`nano_nccl_b200.ops.embedding`."""

    def forward(self, tokens):
        return ops.embedding(tokens, self.weight)


def _modules(checkpoints):
    return (torch.nn.Linear, torch.nn.GELU) if checkpoints is None else (_Linear8, _Gelu8)


class _Attention(torch.nn.Module):
    """Self-attention whose queries and keys are turned by their positions (``rotary``), after a norm of each head where ``qk_norm`` says so.
    Projections keep their inputs in 8 bits where ``checkpoints`` says so; so do the norms."""

    def __init__(self, hidden, heads, rotary, qk_norm, checkpoints):
        super().__init__()
        self.heads, self.rotary, self.checkpoints = heads, rotary, checkpoints
        linear, _ = _modules(checkpoints)
        self.c_attn = linear(hidden, 3 * hidden)
        self.c_proj = linear(hidden, hidden)
        if qk_norm:
            self.q_norm = torch.nn.Parameter(torch.ones(hidden // heads))
            self.k_norm = torch.nn.Parameter(torch.ones(hidden // heads))
        self.qk_norm = qk_norm
        self._frequencies = None  # (not a buffer: it stays in 64 bits whatever type the module is cast to)

    def frequencies(self, device):
        if self._frequencies is None or self._frequencies.device != device:
            rotated = self.c_proj.in_features // self.heads if self.rotary else 0
            self._frequencies = ops.rotary_frequencies(rotated, device=device)[0] if rotated else torch.empty(0, dtype=torch.float64, device=device)
        return self._frequencies

    def forward(self, x):
        b, t, hidden = x.shape
        q, k, v = (p.view(b, t, self.heads, -1) for p in self.c_attn(x).split(hidden, -1))
        positions = torch.arange(t, device=x.device)
        if self.qk_norm:
            q, k = ops.qk_norm_rotary(q, k, self.q_norm, self.k_norm, positions, self.frequencies(x.device), keep=self.checkpoints)
        elif self.rotary:
            q, k = ops.rotary(q, k, positions, self.frequencies(x.device))
        y = torch.nn.functional.scaled_dot_product_attention(q.transpose(1, 2), k.transpose(1, 2), v.transpose(1, 2))
        return self.c_proj(y.transpose(1, 2).reshape(b, t, hidden))


class _Block(torch.nn.Module):
    def __init__(self, hidden, heads, rotary=False, qk_norm=False, checkpoints=None):
        super().__init__()
        linear, gelu = _modules(checkpoints)
        self.plain_attention = not rotary and not qk_norm and checkpoints is None
        self.ln_1 = torch.nn.LayerNorm(hidden)
        self.attn = (torch.nn.MultiheadAttention(hidden, heads, batch_first=True) if self.plain_attention
                     else _Attention(hidden, heads, rotary, qk_norm, checkpoints))
        self.ln_2 = torch.nn.LayerNorm(hidden)
        self.mlp = torch.nn.Sequential(linear(hidden, 4 * hidden), gelu(), linear(4 * hidden, hidden))

    def forward(self, x):
        h = self.ln_1(x)
        x = x + (self.attn(h, h, h, need_weights=False)[0] if self.plain_attention else self.attn(h))
        return x + self.mlp(self.ln_2(x))


# What a model is asked for beside its logits is looked at in functions of their own, which torch.fx keeps as calls: a traced model decides when it is called.
@torch.fx.wrap
def _check_ends(vocabulary, targets, teacher):
    if targets is not None and teacher is not None:
        raise ValueError("targets or a teacher, not both")
    if teacher is not None and vocabulary != "fused":
        raise ValueError("a teacher needs vocabulary='fused'")


@torch.fx.wrap
def _end(x, weight, vocabulary, targets, teacher, temperature):
    _check_ends(vocabulary, targets, teacher)
    if teacher is not None:
        return ops.linear_distillation(x, weight, *teacher, temperature=temperature)
    if targets is not None and vocabulary == "fused":
        return ops.linear_cross_entropy(x, weight, targets)
    logits = x @ weight.t()
    if targets is None:
        return logits
    losses = torch.nn.functional.cross_entropy(logits.flatten(0, -2).float(), targets.flatten().long().clamp(min=-1), ignore_index=-1, reduction="sum")
    return losses / (targets >= 0).sum().clamp(min=1)


class TinyGPT2(torch.nn.Module):
    """``positions``: "learned" (an embedding) or "rotary" (queries and keys are turned). ``qk_norm``: a norm of each head of queries and keys.
    ``checkpoints``: "int8" keeps the inputs of projections, activations and head norms in 8 bits for the backward pass, None keeps them as they
    are. ``vocabulary``: "fused" looks tokens up, and makes losses, without logits in memory (:mod:`nano_nccl_b200.ops.vocabulary`; negative tokens are padding),
    "plain" by torch's own. All but the defaults run on CUDA only (:mod:`nano_nccl_b200.ops`)."""

    vocabulary = "plain"  # of modules that were pickled before there was a choice

    def __init__(self, vocab=512, context=64, hidden=64, layers=2, heads=4, positions="learned", qk_norm=False, checkpoints=None, vocabulary="plain"):
        super().__init__()
        if positions not in ("learned", "rotary"):
            raise ValueError(f"unknown kind of positions '{positions}'")
        if checkpoints not in (None, "int8"):
            raise ValueError(f"unknown kind of checkpoints '{checkpoints}'")
        if vocabulary not in ("plain", "fused"):
            raise ValueError(f"unknown kind of vocabulary '{vocabulary}'")
        if hidden % heads and (positions == "rotary" or qk_norm or checkpoints is not None):
            raise ValueError(f"{heads} heads do not make {hidden}")
        if (positions == "rotary" or qk_norm) and ((hidden // heads) % 2 or hidden // heads > 256):
            raise ValueError(f"{heads} heads of an even size up to 256 do not make {hidden}")
        self.vocabulary = vocabulary
        self.wte = (_Embedding if vocabulary == "fused" else torch.nn.Embedding)(vocab, hidden)
        self.wpe = torch.nn.Embedding(context, hidden) if positions == "learned" else None
        self.blocks = torch.nn.ModuleList([_Block(hidden, heads, positions == "rotary", qk_norm, checkpoints) for _ in range(layers)])
        self.ln_f = torch.nn.LayerNorm(hidden)

    def forward(self, tokens, targets=None, teacher=None, temperature=1.0):
        """Logits; with ``targets`` [batch, tokens] their mean cross entropy (negative targets do not count), with ``teacher``, a pair of the largest
        logits of a teacher and their tokens ([batch, tokens, entries] each), the mean divergence from it (:func:`nano_nccl_b200.ops.linear_distillation`)."""
        _check_ends(self.vocabulary, targets, teacher)
        x = self.wte(tokens)
        if self.wpe is not None:
            x = x + self.wpe(torch.arange(tokens.shape[1], device=tokens.device))
        for b in self.blocks:
            x = b(x)
        return _end(self.ln_f(x), self.wte.weight, self.vocabulary, targets, teacher, temperature)
