"""Torch custom ops (``torch.ops.b200ccl.*``) over a registered communicator.

The ops take a communicator id instead of an object so that they can be traced and captured like
any other op. ``register_communicator`` returns the id; id 0 is the default communicator set by
``set_default_communicator``.

Beside them, the operators of a training step that run on one GPU and need no communicator: activations kept
in 8 bits for the backward pass (``checkpoint8``) and the rotation and norm of queries and keys (``rotation``).
"""
from .checkpoint8 import Packed8, check_async_error, gelu8, linear8, pack8, unpack8, weight_grad8  # noqa: F401
from .collectives import (all_gather, all_reduce, all_reduce_, get_communicator, reduce_scatter,  # noqa: F401
                          register_communicator, set_default_communicator)
from .rotation import qk_norm_rotary, rotary, rotary_frequencies  # noqa: F401
