"""LayerNorm, dropout from a counter-based generator, and both in one pass with the activation before them
(include/amber_mpn.h: amber_mpn_tail_forward / _backward, amber_mpn_keep_mask, amber_mpn_generator_take).  GPU tensors only:
there is no CPU path.

    gen = CounterGenerator(seed, device="cuda")          # an nn.Module: (seed, offset) in a device buffer
    state = gen.take()                                   # int64[2], one range of random numbers; no synchronisation
    y = layer_norm(x, weight, bias)
    y = dropout(x, 0.1, state)                           # the mask is never stored: the backward pass draws it again
    y = activate_norm_dropout(z, "leakyrelu", weight, bias, p=0.1, state=state)   # what follows a Linear of the decoder
    keep = keep_mask(num_edges, 0.1, state)

Element i (row-major) of a call owns word i & 3 of Philox-4x32-10 under key `seed` at counter (i >> 2, offset + sequence); it is
dropped iff the word is below floor(p 2^32).  A dropped element is +0 whatever it held, and so is the gradient that reaches its place
(x's own gradient there, unless a norm stands between: its gradient joins the whole row).

Types: float32, bfloat16, float16; weight and bias in x's type or float32.  Sums, statistics and activations are float32,
rounded once at the end.  Rows are the last dimension; rows that are evenly spaced with adjacent features are read in place,
anything else is copied first.  First derivatives only.

Inside a HIP graph: `take` and the operators may be captured; the generator's state lives on the device, so every replay draws
new numbers.  Capturing a backward pass follows torch's own rule: no autograd graph that was recorded outside the capture may
still hold the same leaves.

Recomputing (torch.utils.checkpoint): call `take` outside the recomputed function and hand its result in; a `take` that is run
again draws other numbers.
"""
from __future__ import annotations

from typing import Optional

import torch
from torch import nn

from . import _lib

_tail = None  # the binding's entry, looked up once: a short call's time is mostly the host's


def _run(x, weight, bias, state, activation: int, normalize: bool, p: float, eps: float, sequence: int) -> torch.Tensor:
    global _tail
    if _tail is None:
        _tail = _lib.binding().tail
    return _tail(x, weight, bias, state, activation, normalize, p, eps, sequence)


def _signed(value: int) -> int:
    value = int(value) & (1 << 64) - 1
    return value - (1 << 64) if value >> 63 else value


class CounterGenerator(nn.Module):
    """(seed, offset) of the counter-based generator in a device buffer (not part of a state_dict: get_state / set_state).
    Two generators with one seed draw the same numbers: ranks that see different data should get different seeds."""

    def __init__(self, seed: Optional[int] = None, device=None):
        super().__init__()
        if seed is None:
            seed = torch.initial_seed()
        self.register_buffer("state", torch.tensor([_signed(seed), 0], dtype=torch.int64, device=device), persistent=False)

    def take(self, count: int = 1) -> torch.Tensor:
        """The next `count` ranges: int64[2] (seed, offset), to be used with sequence = 0 .. count - 1."""
        return _lib.binding().generator_take(self.state, count)

    def get_state(self):
        """(seed, offset) as Python ints (reads the device)."""
        seed, offset = self.state.tolist()
        return seed & (1 << 64) - 1, offset & (1 << 64) - 1

    def set_state(self, seed: int, offset: int = 0) -> None:
        self.state.copy_(torch.tensor([_signed(seed), _signed(offset)], dtype=torch.int64))

    def extra_repr(self) -> str:
        return f"device={self.state.device}"


def keep_mask(count: int, p: float, state: torch.Tensor, sequence: int = 0) -> torch.Tensor:
    """bool[count]: the elements that the generator keeps with probability 1 - p."""
    return _lib.binding().keep_mask(count, p, state, sequence)


def layer_norm(x: torch.Tensor, weight: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None,
               eps: float = 1e-5) -> torch.Tensor:
    """(x - mean) / sqrt(var + eps) * weight + bias over the last dimension (torch.nn.functional.layer_norm with one
    normalised dimension), differentiable with respect to all three."""
    return _run(x, weight, bias, None, _lib.ACT_NONE, True, 0.0, eps, 0)


def dropout(x: torch.Tensor, p: float, state: Optional[torch.Tensor] = None, *, sequence: int = 0, training: bool = True) -> torch.Tensor:
    """x / (1 - p) where the generator keeps an element, 0 elsewhere; x itself for p = 0 or training = False."""
    return _run(x, None, None, state, _lib.ACT_NONE, False, p if training else 0.0, 0.0, sequence)


def activate_norm_dropout(x: torch.Tensor, activation: Optional[str], weight: Optional[torch.Tensor] = None,
                          bias: Optional[torch.Tensor] = None, *, normalize: bool = True, eps: float = 1e-5, p: float = 0.0,
                          state: Optional[torch.Tensor] = None, sequence: int = 0, training: bool = True) -> torch.Tensor:
    """dropout(layer_norm(act(x))) in one pass over x, and one over x and the gradient in the backward pass; without
    `normalize` dropout(act(x)).  activation: a name of the decoder's activations (relu, leakyrelu, tanh, elu, silu / swish,
    mish, gelu) or None."""
    act = _lib.ACT_NONE
    if activation is not None:
        act = _lib.ACT.get(activation.lower(), None)
        if act is None:
            raise ValueError(f"Unknown activation function '{activation}'")
    return _run(x, weight, bias, state, act, normalize, p if training else 0.0, eps, sequence)
