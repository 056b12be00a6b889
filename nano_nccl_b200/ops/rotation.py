"""Queries and keys turned by their positions, alone or in the same pass as the norm of each head.

``q`` and ``k`` are [tokens, heads, dim] or [batch, tokens, heads, dim], with any strides but on the last axis (a view into the output of a
joint projection costs no copy); their heads may differ in number, and either may be None. ``positions`` is [tokens] or
[batch, tokens], int64 or int32. ``frequencies`` is a float64 vector, radians per position of each pair; it turns the first
``2 * len(frequencies)`` elements of a head and leaves the others as they are. The pairs are ``(i, i + len(frequencies))``
(layout ``"half"``) or ``(2i, 2i + 1)`` (``"interleaved"``). Angles are made in 64 bits, so positions may be far
(an error of 2e-7, and beyond 2^26 turns of 2^-49 radians for each turn).
"""
import math

import torch

from .._lib import load_native_calls

_LAYOUTS = {"half": False, "interleaved": True}


def rotary_frequencies(rotated, base=10000.0, scaling=None, factor=1.0, context=None, fast=32.0, slow=1.0, device="cuda"):
    """(frequencies, magnitude) of ``rotated`` elements of a head: ``base ** (-2i / rotated)`` radians per position, and 1.

    ``scaling`` stretches them for contexts ``factor`` times as long as the ``context`` positions of the training:

    * ``"linear"``: every frequency divided by ``factor`` (positions interpolated);
    * ``"ntk"``: a larger base, ``base * factor ** (rotated / (rotated - 2))``, which divides the slowest frequency by ``factor`` and leaves the fastest;
    * ``"yarn"``: pairs that make more than ``fast`` turns in ``context`` positions stay, those that make fewer than ``slow`` are divided by
      ``factor``, with a line between by pair index; magnitude ``0.1 ln(factor) + 1``.
    """
    if rotated < 2 or rotated % 2:
        raise ValueError("the rotated part must be even and at least 2")
    if base <= 1.0 or factor < 1.0:
        raise ValueError("base must be above 1 and factor at least 1")
    pairs = torch.arange(rotated // 2, dtype=torch.float64)
    magnitude = 1.0
    if scaling == "ntk":
        if rotated == 2:
            raise ValueError("scaling 'ntk' needs more than one pair")
        base = base * factor ** (rotated / (rotated - 2))
    frequencies = base ** (-2.0 * pairs / rotated)
    if scaling == "linear":
        frequencies = frequencies / factor
    elif scaling == "yarn":
        if context is None or context < 1 or not fast > slow > 0:
            raise ValueError("scaling 'yarn' needs the context of the training, and fast > slow > 0")
        # The pair index that makes n turns in `context` positions.
        pair_of = lambda n: rotated * math.log(context / (2.0 * math.pi * n)) / (2.0 * math.log(base))  # noqa: E731
        low, high = math.floor(pair_of(fast)), math.ceil(pair_of(slow))
        divided = ((pairs - low) / (high - low)).clamp(0.0, 1.0)
        frequencies = frequencies * (1.0 - divided) + frequencies / factor * divided
        magnitude = 0.1 * math.log(factor) + 1.0
    elif scaling not in (None, "ntk"):
        raise ValueError(f"unknown scaling '{scaling}'")
    return frequencies.to(device), magnitude


def _interleaved(layout):
    if layout not in _LAYOUTS:
        raise ValueError(f"unknown layout '{layout}'")
    return _LAYOUTS[layout]


def rotary(q, k, positions, frequencies, layout="half", magnitude=1.0):
    """(q, k) turned by their positions: ``magnitude * (u cos - v sin, u sin + v cos)`` for every pair, one rounding at the end."""
    return load_native_calls().rotary(q, k, positions, frequencies, _interleaved(layout), magnitude)


def qk_norm_rotary(q, k, q_weight, k_weight, positions, frequencies, layout="half", magnitude=1.0, eps=1e-6, keep=None):
    """(q, k) after the norm of each head, ``x * (mean(x^2) + eps)^(-1/2) * weight``, and the rotation of :func:`rotary`, in one pass.

    ``q_weight`` and ``k_weight``: [dim], of the same dtype. For the backward pass q and k are kept as they are, or, with ``keep="int8"``,
    in 8 bits, as in :mod:`.checkpoint8`, a head of a token being one block: the gradients are then those of the formula at what was kept. Under autocast, weights of another dtype are
    cast to that of q and k."""
    interleaved = _interleaved(layout)
    if keep not in (None, "int8"):
        raise ValueError(f"unknown way to keep queries and keys '{keep}'")
    if not eps >= 0.0:
        raise ValueError("eps must not be negative")
    if torch.is_autocast_enabled("cuda"):
        q_weight, k_weight = (w if x is None or w is None else w.to(x.dtype) for x, w in ((q, q_weight), (k, k_weight)))
    return load_native_calls().qk_norm_rotary(q, k, q_weight, k_weight, positions, frequencies, interleaved, magnitude, eps, keep == "int8")
