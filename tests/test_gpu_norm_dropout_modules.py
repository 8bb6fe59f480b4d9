"""LayerNorm / dropout operators on the GPU: accuracy of long sums, of constant rows and of the activations' tails, dropped places'
gradients, and the framework's own modules over the operators (recomputation, changed modules, hooks).  Needs an MI355X: `-m gpu`.

Tolerances: u = 2^-24, half a step of fp32; a row's sum adds at most 48 terms in a row whatever its width (a lane's at most 16 elements, or
a sum that carries its rounding errors along, then a tree), a sum over rows at most `chain`."""
import math

import pytest
import torch
import torch.utils.checkpoint

from amber_amd import norm_dropout as nd, synthetic as syn
from amber_amd.architecture.mlp import MLP
from amber_amd.architecture.supervised_mpn import SupervisedMPN
from amber_amd.config import AttrDict, default_architecture
from oracle import norm_dropout_oracle as orc
from test_gpu_norm_dropout import ACTS, DTYPES, U, _compare, _data, _decoder, _half, _run, _state

pytestmark = pytest.mark.gpu
DEPTH = 48


def _norm_bounds(x, w, b, go, chain, eps=1e-5):
    """Error bounds of layer_norm's (y, dx, dw, db) in fp32: the two means, the variance and the backward pass's two means within DEPTH u of
    their absolute terms, a few u for each product; the mean that the backward pass reads is rounded once, which moves its n by
    u |mean| rstd."""
    x, w, b, g = (t.double() for t in (x, w, b, go))
    mean = x.mean(1, keepdim=True)
    d = x - mean
    rstd = 1 / torch.sqrt((d * d).mean(1, keepdim=True) + eps)
    n = d * rstd
    # the first mean is off by DEPTH u mean|x|; the differences' own mean takes that off, to DEPTH u of mean|d|
    dm = DEPTH * U * d.abs().mean(1, keepdim=True) + (DEPTH * U) ** 2 * x.abs().mean(1, keepdim=True)
    dr = (DEPTH + 6) * U
    dn = rstd * (dm + 2 * U * d.abs()) + n.abs() * dr
    y = n * w + b
    by = w.abs() * dn + 4 * U * ((n * w).abs() + b.abs()) + U * y.abs()
    dn = dn + U * mean.abs() * rstd
    h = g * w
    m0, m1 = h.mean(1, keepdim=True), (h * n).mean(1, keepdim=True)
    dm0 = DEPTH * U * h.abs().mean(1, keepdim=True)
    dm1 = DEPTH * U * (h * n).abs().mean(1, keepdim=True) + (h.abs() * dn).mean(1, keepdim=True)
    q = h - m0 - n * m1
    dq = U * h.abs() + dm0 + n.abs() * dm1 + dn * m1.abs() + 4 * U * (h.abs() + m0.abs() + (n * m1).abs())
    bx = rstd * dq + (rstd * q).abs() * (dr + 4 * U)
    bw = chain * U * (g * n).abs().sum(0) + (g.abs() * dn).sum(0)
    bb = chain * U * g.abs().sum(0)
    return [1.01 * t for t in (by, bx, bw, bb)]


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("act", [None] + ACTS)
def test_gradients_of_dropped_places_are_plus_zero(gpu_device, act, dtype):
    """Without the norm the gradient of a dropped place is +0 whatever x and the incoming gradient hold there: x where the
    activation's derivative is negative, NaN or 0 times infinity, a gradient that is negative, infinite or NaN."""
    state, t = _state(gpu_device), DTYPES[dtype]
    values = torch.tensor([-1.5, -4.0, 2.0, -0.0, float("nan"), float("inf"), float("-inf")])
    x = values.repeat(331)[:2310].view(33, 70).to(t).to(gpu_device).requires_grad_()
    keep = nd.keep_mask(x.numel(), 0.5, state).view(x.shape)
    for grad in (1.0, -1.0, float("inf"), float("nan")):
        y = nd.activate_norm_dropout(x, act, normalize=False, p=0.5, state=state)
        g, = torch.autograd.grad(y, x, torch.full_like(x, grad))
        assert not bool(g[~keep].any()) and not bool(torch.signbit(g[~keep]).any())  # NaN counts as true
        if grad == 1.0:
            assert bool(torch.isfinite(g[keep & (x.abs() <= 4.0)]).all())
