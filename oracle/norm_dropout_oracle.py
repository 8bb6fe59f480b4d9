"""CPU restatement in float64 of activation -> LayerNorm -> dropout with its gradients, and of the counter-based generator
(Philox-4x32-10, Salmon, Moraes, Dror, Shaw: Parallel random numbers, as easy as 1, 2, 3; SC 2011).  Test infrastructure only.

The layers are those of the decoder MLP (src/algorithm/architecture/mlp.py:58-96)."""
import numpy as np
import torch


def philox(counter, key):
    """counter: uint32 [..., 4], key: (k0, k1) -> uint32 [..., 4]"""
    c = [np.asarray(counter)[..., i].astype(np.uint64) for i in range(4)]
    k0, k1 = int(key[0]), int(key[1])
    low = np.uint64(0xFFFFFFFF)
    shift = np.uint64(32)
    for _ in range(10):
        p0, p1 = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        c = [(p1 >> shift) ^ c[1] ^ np.uint64(k0), p1 & low, (p0 >> shift) ^ c[3] ^ np.uint64(k1), p0 & low]
        k0, k1 = (k0 + 0x9E3779B9) & 0xFFFFFFFF, (k1 + 0xBB67AE85) & 0xFFFFFFFF
    return np.stack(c, axis=-1).astype(np.uint32)


def words(start, count, seed, offset):
    """The words of elements start .. start + count - 1 (uint32)."""
    seed, offset = seed & (1 << 64) - 1, offset & (1 << 64) - 1
    first, last = start // 4, (start + count + 3) // 4
    group = np.arange(first, last, dtype=np.uint64)
    ctr = np.stack([group & np.uint64(0xFFFFFFFF), group >> np.uint64(32), np.full_like(group, offset & 0xFFFFFFFF),
                    np.full_like(group, offset >> 32)], axis=-1)
    w = philox(ctr, (seed & 0xFFFFFFFF, seed >> 32)).reshape(-1)
    return w[start - 4 * first:start - 4 * first + count]


def keep(count, p, seed, offset, start=0):
    return torch.from_numpy(words(start, count, seed, offset).astype(np.int64) >= int(p * 2.0 ** 32))


def act(x, name):
    f = torch.nn.functional
    return {None: lambda t: t, "relu": torch.relu, "leakyrelu": lambda t: f.leaky_relu(t, 0.01), "tanh": torch.tanh, "elu": f.elu,
            "silu": f.silu, "swish": f.silu, "mish": f.mish, "gelu": f.gelu}[name](x)


def tail(x, activation=None, weight=None, bias=None, normalize=True, eps=1e-5, kept=None, p=0.0, grad=None):
    """(y,) or (y, dx[, dweight][, dbias]) in float64.  kept: bool like x, or None (no dropout)."""
    leaves = [t.detach().double().requires_grad_(grad is not None) for t in (x, weight, bias) if t is not None]
    rest = leaves[1:]
    y = act(leaves[0], activation)
    if normalize:
        d = y - y.mean(-1, keepdim=True)
        y = d / torch.sqrt((d * d).mean(-1, keepdim=True) + eps)
        if weight is not None:
            y = y * rest.pop(0)
        if bias is not None:
            y = y + rest.pop(0)
    if kept is not None:
        y = torch.where(kept, y * (1.0 / (1.0 - p) if p < 1.0 else 0.0), torch.zeros_like(y))
    if grad is None:
        return (y,)
    return (y.detach(),) + torch.autograd.grad(y, leaves, grad.double())
