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
dropped iff the word is below floor(p 2^32).  A dropped element is +0 whatever it held, and so is its gradient.

Types: float32, bfloat16, float16; weight and bias in x's type or float32.  Sums, statistics and activations are float32,
rounded once at the end.  Rows are the last dimension; rows that are evenly spaced with adjacent features are read in place,
anything else is copied first.  First derivatives only.

Inside a HIP graph: `take` and the operators may be captured; the generator's state lives on the device, so every replay draws
new numbers.  Capturing a backward pass follows torch's own rule: no autograd graph that was recorded outside the capture may
still hold the same leaves.
"""
from __future__ import annotations

import ctypes as C
import functools
from typing import Optional

import torch
from torch import nn
from torch.autograd.function import once_differentiable

from . import _lib
from .csr import _require_cuda

_DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}


def _check_p(p: float) -> float:
    if not 0.0 <= p <= 1.0:
        raise ValueError(f"Dropout probability has to be between 0 and 1 (got {p})")
    return float(p)


def _check_state(state: Optional[torch.Tensor], device) -> torch.Tensor:
    if state is None:
        raise ValueError("amber_amd: dropout needs the generator's `state` (CounterGenerator.take())")
    if state.dtype != torch.int64 or tuple(state.shape) != (2,) or not state.is_contiguous():
        raise ValueError(f"amber_amd: `state` must be a contiguous int64 tensor (seed, offset), got {state.dtype} {tuple(state.shape)}")
    if state.device != device:
        raise ValueError(f"amber_amd: `state` is on {state.device}, the data on {device}")
    return state


def _check_sequence(sequence: int) -> int:
    if not 0 <= sequence < 1 << 62:
        raise ValueError(f"amber_amd: sequence has to be between 0 and 2**62 (got {sequence})")
    return int(sequence)


def _call(name: str, device, *args) -> None:
    """One library call on `device`'s current stream."""
    fn = getattr(_lib.load(), name)
    stream = torch.cuda.current_stream(device).cuda_stream
    if device.index == torch.cuda.current_device():
        rc = fn(*args, stream)
    else:
        with torch.cuda.device(device):
            rc = fn(*args, stream)
    if rc:
        _lib.check(rc, name)


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
        if not 1 <= count < 1 << 62:
            raise ValueError(f"amber_amd: take of {count} ranges")
        _require_cuda(self.state, "generator state")
        taken = torch.empty_like(self.state)
        _call("amber_mpn_generator_take", self.state.device, self.state.data_ptr(), int(count), taken.data_ptr())
        return taken

    def get_state(self):
        """(seed, offset) as Python ints (reads the device)."""
        seed, offset = self.state.tolist()
        return seed & (1 << 64) - 1, offset & (1 << 64) - 1

    def set_state(self, seed: int, offset: int = 0) -> None:
        self.state.copy_(torch.tensor([_signed(seed), _signed(offset)], dtype=torch.int64))

    def extra_repr(self) -> str:
        return f"device={self.state.device}"


def _signed(value: int) -> int:
    value = int(value) & (1 << 64) - 1
    return value - (1 << 64) if value >> 63 else value


def keep_mask(count: int, p: float, state: torch.Tensor, sequence: int = 0) -> torch.Tensor:
    """bool[count]: the elements that the generator keeps with probability 1 - p."""
    if count < 0:
        raise ValueError(f"amber_amd: a mask of {count} elements")
    p = _check_p(p)
    if isinstance(state, torch.Tensor):
        _require_cuda(state, "state")
    _check_state(state, getattr(state, "device", None))
    out = torch.empty(count, dtype=torch.bool, device=state.device)
    _call("amber_mpn_keep_mask", state.device, state.data_ptr(), _check_sequence(sequence), p, int(count), out.data_ptr())
    return out


@functools.lru_cache(maxsize=512)
def _desc(dtype, weight_dtype, activation: int, normalize: bool, p: float, eps: float, sequence: int):
    desc = _lib.AmberTailDesc(dtype=_DTYPES[dtype], weight_dtype=_DTYPES[weight_dtype], activation=activation,
                              normalize=int(normalize), p=p, eps=eps, sequence=sequence)
    return desc, C.byref(desc)


def _rows(t: torch.Tensor, width: int, dense: bool):
    """(tensor that owns the memory, row stride): evenly spaced rows of adjacent features, a copy where t is not that."""
    if t.is_contiguous():
        return t, width
    if not dense and width > 0:
        r = t
        if t.dim() != 2:
            r = t.reshape(-1, width)  # a view where one stride covers the leading dimensions
        if width == 1 or r.stride(1) == 1:
            return r, (r.stride(0) if r.shape[0] > 1 else width)
    return t.contiguous(), width


class _Tail(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, state, key):
        y, xr, ldx, stats = _forward(x, weight, bias, state, key, True)
        needs_x = key[3] or key[2] != _lib.ACT_NONE
        ctx.save_for_backward(xr if needs_x else None, weight, stats, state)
        ctx.key, ctx.ldx, ctx.shape, ctx.has_bias = key, ldx, x.shape, bias is not None
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_y):
        x, weight, stats, state = ctx.saved_tensors
        key, shape = ctx.key, ctx.shape
        normalize = key[3]
        width = shape[-1] if len(shape) else 1
        rows = grad_y.numel() // width if width else 0
        g, ldg = _rows(grad_y, width, not normalize)
        dev = grad_y.device
        need_x, need_w, need_b = ctx.needs_input_grad[:3]
        grad_x = torch.empty(shape, dtype=grad_y.dtype, device=dev) if need_x else None
        grad_w = grad_b = ws = None
        ws_bytes = 0
        desc, ref = _desc(*key)
        if need_w or need_b:
            if need_w:
                grad_w = torch.empty(width, dtype=key[1], device=dev)
            if need_b:
                grad_b = torch.empty(width, dtype=key[1], device=dev)
            ws_bytes = _lib.load().amber_mpn_tail_backward_workspace_bytes(ref, rows, width)
            if ws_bytes == 0:
                _lib.check(-1, "amber_mpn_tail_backward_workspace_bytes")
            ws = torch.empty(ws_bytes, dtype=torch.uint8, device=dev)
        ptr = _lib.ptr
        _call("amber_mpn_tail_backward", dev, ref, rows, width, ptr(x), ctx.ldx, g.data_ptr(), ldg, ptr(weight), ptr(stats), ptr(state),
              ptr(grad_x), ptr(grad_w), ptr(grad_b), ptr(ws), ws_bytes)
        return grad_x, grad_w, grad_b, None, None


def _forward(x, weight, bias, state, key, train: bool):
    normalize = key[3]
    width = x.shape[-1] if x.dim() else 1
    rows = x.numel() // width if width else 0
    xr, ldx = _rows(x, width, not normalize)
    y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    stats = torch.empty(2 * rows, dtype=torch.float32, device=x.device) if normalize and train else None
    ptr = _lib.ptr
    _call("amber_mpn_tail_forward", x.device, _desc(*key)[1], rows, width, xr.data_ptr(), ldx, ptr(weight), ptr(bias), ptr(state),
          y.data_ptr(), ptr(stats))
    return y, xr, ldx, stats


def _apply(x, weight, bias, state, key):
    if torch.is_grad_enabled() and (x.requires_grad or (weight is not None and weight.requires_grad)
                                    or (bias is not None and bias.requires_grad)):
        return _Tail.apply(x, weight, bias, state, key)
    return _forward(x, weight, bias, state, key, False)[0]


def _check_input(x: torch.Tensor) -> None:
    _require_cuda(x, "x")
    if x.dtype not in _DTYPES:
        raise TypeError(f"amber_amd: x must be float32, bfloat16 or float16, got {x.dtype}")


def _check_weights(x: torch.Tensor, weight: Optional[torch.Tensor], bias: Optional[torch.Tensor]):
    """(weight, bias, their common type)"""
    if x.dim() == 0 or x.shape[-1] == 0:
        raise ValueError(f"amber_amd: LayerNorm over the last dimension of a tensor of shape {tuple(x.shape)}")
    wdtype = None
    for name, t in (("weight", weight), ("bias", bias)):
        if t is None:
            continue
        if tuple(t.shape) != (x.shape[-1],):
            raise ValueError(f"amber_amd: {name} of shape {tuple(t.shape)} for {x.shape[-1]} features")
        if t.device != x.device:
            raise ValueError(f"amber_amd: {name} is on {t.device}, x on {x.device}")
        if t.dtype != x.dtype and t.dtype != torch.float32:
            raise TypeError(f"amber_amd: {name} must be of x's type ({x.dtype}) or float32, got {t.dtype}")
        if wdtype is not None and t.dtype != wdtype:
            raise TypeError(f"amber_amd: weight is {wdtype}, bias {t.dtype}")
        wdtype = t.dtype
    return (weight if weight is None else weight.contiguous()), (bias if bias is None else bias.contiguous()), wdtype or x.dtype


def _check_eps(eps: float) -> float:
    if not 0.0 <= eps < 3.0e38:
        raise ValueError(f"amber_amd: eps must be finite and not negative (got {eps})")
    return float(eps)


def layer_norm(x: torch.Tensor, weight: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None,
               eps: float = 1e-5) -> torch.Tensor:
    """(x - mean) / sqrt(var + eps) * weight + bias over the last dimension (torch.nn.functional.layer_norm with one
    normalised dimension), differentiable with respect to all three."""
    _check_input(x)
    weight, bias, wdtype = _check_weights(x, weight, bias)
    return _apply(x, weight, bias, None, (x.dtype, wdtype, _lib.ACT_NONE, True, 0.0, _check_eps(eps), 0))


def dropout(x: torch.Tensor, p: float, state: Optional[torch.Tensor] = None, *, sequence: int = 0, training: bool = True) -> torch.Tensor:
    """x / (1 - p) where the generator keeps an element, 0 elsewhere; x itself for p = 0 or training = False."""
    _check_input(x)
    p = _check_p(p)
    if not training or p == 0.0:
        return x
    return _apply(x, None, None, _check_state(state, x.device),
                  (x.dtype, x.dtype, _lib.ACT_NONE, False, p, 0.0, _check_sequence(sequence)))


def activate_norm_dropout(x: torch.Tensor, activation: Optional[str], weight: Optional[torch.Tensor] = None,
                          bias: Optional[torch.Tensor] = None, *, normalize: bool = True, eps: float = 1e-5, p: float = 0.0,
                          state: Optional[torch.Tensor] = None, sequence: int = 0, training: bool = True) -> torch.Tensor:
    """dropout(layer_norm(act(x))) in one pass over x, and one over x and the gradient in the backward pass; without
    `normalize` dropout(act(x)).  activation: a name of the decoder's activations (relu, leakyrelu, tanh, elu, silu / swish,
    mish, gelu) or None."""
    _check_input(x)
    key = activation.lower() if isinstance(activation, str) else activation
    if key is not None and key not in _lib.ACT:
        raise ValueError(f"Unknown activation function '{activation}'")
    act = _lib.ACT_NONE if key is None else _lib.ACT[key]
    p = _check_p(p)
    if not training:
        p = 0.0
    if p > 0.0:
        _check_state(state, x.device)
    else:
        state = None
    sequence = _check_sequence(sequence)
    if normalize:
        weight, bias, wdtype = _check_weights(x, weight, bias)
        eps = _check_eps(eps)
    else:
        if weight is not None or bias is not None:
            raise ValueError("amber_amd: weight / bias without normalize")
        wdtype, eps = x.dtype, 0.0
        if act == _lib.ACT_NONE and p == 0.0:
            return x
    return _apply(x, weight, bias, state, (x.dtype, wdtype, act, bool(normalize), p, eps, sequence if p > 0.0 else 0))
