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

Recomputing (torch.utils.checkpoint): a `take` that is run again draws other numbers.  Call it outside the recomputed function and hand
its result in, or have the recomputation take the same ranges:

    checkpoint(function, x, use_reentrant=False, context_fn=gen.checkpoint_contexts)

The framework's own modules (decoder layers, edge dropout) take ranges inside their forward and refuse to do so anew in a backward pass.
"""
from __future__ import annotations

import threading
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


_thread = threading.local()  # .contexts: the _Recorded / _Replayed that are open on this thread, the innermost last


def _take(generator, count: int, depth: Optional[int] = None) -> torch.Tensor:
    """The next `count` ranges as the innermost of the first `depth` open contexts has them, or the generator itself."""
    contexts = getattr(_thread, "contexts", ())
    for i in range(len(contexts) if depth is None else depth, 0, -1):
        if contexts[i - 1].generator is generator:
            return contexts[i - 1].take(count, i - 1)
    return _lib.binding().generator_take(generator.state, count)


class _Recorded:
    """While open: what is taken from the generator is kept in `taken`."""

    def __init__(self, generator, taken: list):
        self.generator, self.taken = generator, taken

    def __enter__(self):
        if not hasattr(_thread, "contexts"):
            _thread.contexts = []
        _thread.contexts.append(self)

    def __exit__(self, *exc):
        _thread.contexts.pop()

    def take(self, count: int, depth: int) -> torch.Tensor:
        state = _take(self.generator, count, depth)  # a checkpoint inside a recomputed one records what that one replays
        self.taken.append((count, state))
        return state


class _Replayed(_Recorded):
    """While open: the ranges of `taken` once more, in their order."""

    def __enter__(self):
        super().__enter__()
        self.next = 0

    def take(self, count: int, depth: int) -> torch.Tensor:
        if self.next >= len(self.taken) or self.taken[self.next][0] != count:
            raise RuntimeError("amber_amd: the recomputed pass takes other ranges than the first one")
        self.next += 1
        return self.taken[self.next - 1][1]


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
        return _take(self, count)

    def take_in_module(self, count: int = 1) -> torch.Tensor:
        """`take` for a module's forward pass.  Inside a backward pass, where only a recomputation runs it, the ranges of the first pass
        or a RuntimeError: another mask would belong to other gradients."""
        if torch._C._current_graph_task_id() != -1 and not any(isinstance(c, _Replayed) and c.generator is self
                                                               for c in getattr(_thread, "contexts", ())):
            raise RuntimeError("amber_amd: a recomputed forward pass would draw other numbers than the first one; call "
                               "torch.utils.checkpoint.checkpoint with use_reentrant=False and context_fn=generator.checkpoint_contexts")
        return _take(self, count)

    def checkpoint_contexts(self):
        """context_fn of torch.utils.checkpoint.checkpoint(..., use_reentrant=False): a pair of contexts, for the first pass and for its
        recomputations, which take the ranges that the first pass took."""
        taken: list = []
        return _Recorded(self, taken), _Replayed(self, taken)

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
