"""LayerNorm, dropout and activation -> LayerNorm -> dropout on the GPU against the float64 oracle.  Needs an MI355X: `-m gpu`.

Tolerances, elementwise, with u = 2^-24 (half a step of fp32), D the row's width, e the relative half step of the output's type:
  a sum over a row adds at most `depth` = 48 + D / 64 terms in a row (a lane's own elements, then a tree over the lanes), so its
    error is <= depth u sum|terms|; a sum over R rows in any order: <= R u sum|terms|;
  an activation in fp32 is within 4 u |x| + 4 u |a| of its value (gelu and its like multiply x by a factor known to a few u), its
    derivative within 8 u (1 + |x|);
  n = (a - mean) rstd: error dn = rstd (da + depth u mean|a| + u |a - mean|) + |n| dr, dr = (depth + 4) u + the mean's error in the
    variance (its square, negligible) + mean(|d| da) rstd^2;
  y: |w| dn + 4 u (|n w| + |b|), times the dropout's scale, plus e |y|;
  backward: h = g' w; the two means carry depth u of their absolute terms plus what dn brings; dx: rstd |act'| times the sum of these
    plus 4 u of the terms, plus |da| times the derivative's error, plus |dx| dr, plus e |dx|;
  dweight: R u sum|g' n| + sum |g'| dn + e |dw|;  dbias: R u sum|g'| + e |db|.
Everything is bounded by 1.01 of that (second-order terms)."""
import math

import pytest
import torch
import torch.utils.checkpoint

from amber_amd import norm_dropout as nd, synthetic as syn
from amber_amd.architecture.mlp import MLP
from amber_amd.architecture.supervised_mpn import SupervisedMPN
from amber_amd.config import AttrDict, default_architecture
from oracle import norm_dropout_oracle as orc

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
ACTS = ["relu", "leakyrelu", "tanh", "elu", "silu", "mish", "gelu"]
DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}


def _half(t):
    """relative half step of a type (and of its subnormals, absolute)"""
    return torch.finfo(t).eps / 2, torch.finfo(t).smallest_normal * torch.finfo(t).eps


def _data(rows, width, dtype, wdtype, seed, grad=True):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, width, generator=g) * 1.3 + 0.4 * torch.randn(width, generator=g)
    w, b = 1 + 0.3 * torch.randn(width, generator=g), 0.3 * torch.randn(width, generator=g)
    go = torch.randn(rows, width, generator=g) if grad else None
    return x.to(dtype), w.to(wdtype), b.to(wdtype), go.to(dtype) if grad else None


def _bounds(x, act, w, b, normalize, eps, kept, p, go, dtype, wdtype):
    """Error bounds of (y, dx, dw, db), the docstring's formulas in float64."""
    x = x.double()
    rows, width = x.shape
    depth = 48 + width / 64
    xa = x.clone().requires_grad_()
    a = orc.act(xa, act)
    dact, = torch.autograd.grad(a.sum(), xa)
    a = a.detach()
    da = torch.zeros_like(x) if act is None else 4 * U * (x.abs() + a.abs())
    ddact = torch.zeros_like(x) if act in (None, "relu") else 8 * U * (1 + x.abs())
    scale = 1.0 / (1.0 - p) if p < 1 else 0.0
    keep = torch.ones_like(x) if kept is None else kept.double()
    scale = scale if kept is not None else 1.0
    e, tiny = _half(dtype)
    we, wtiny = _half(wdtype)
    gp = None if go is None else go.double() * keep * scale
    dgp = None if gp is None else 2 * U * gp.abs()
    if not normalize:
        y = a * keep * scale
        by = da * keep * scale + 2 * U * y.abs() + e * y.abs() + tiny
        bx = None if gp is None else gp.abs() * ddact + dgp * dact.abs() + 2 * U * (gp * dact).abs() + e * (gp * dact).abs() + tiny
        return [1.01 * t for t in (by, bx) if t is not None]
    w, b = w.double(), b.double()
    mean = a.mean(1, keepdim=True)
    d = a - mean
    rstd = 1 / torch.sqrt((d * d).mean(1, keepdim=True) + eps)
    n = d * rstd
    dm = depth * U * a.abs().mean(1, keepdim=True) + da.mean(1, keepdim=True)
    dr = (depth + 4) * U + (d.abs() * (da + dm)).mean(1, keepdim=True) * rstd ** 2
    dn = rstd * (da + dm + U * d.abs()) + n.abs() * dr
    y = (n * w + b) * keep * scale
    by = keep * scale * (w.abs() * dn + 4 * U * ((n * w).abs() + b.abs())) + e * y.abs() + tiny
    if gp is None:
        return [1.01 * by]
    h = gp * w
    dh = 3 * U * h.abs()
    m0, m1 = h.mean(1, keepdim=True), (h * n).mean(1, keepdim=True)
    dm0 = depth * U * h.abs().mean(1, keepdim=True) + dh.mean(1, keepdim=True)
    dm1 = depth * U * (h * n).abs().mean(1, keepdim=True) + (h.abs() * dn).mean(1, keepdim=True) + (dh * n.abs()).mean(1, keepdim=True)
    q = h - m0 - n * m1
    dq = dh + dm0 + n.abs() * dm1 + dn * m1.abs() + 4 * U * (h.abs() + m0.abs() + (n * m1).abs())
    dx = rstd * q * dact
    bx = rstd * dact.abs() * dq + dx.abs() * (dr + 4 * U) + (rstd * q).abs() * ddact + e * dx.abs() + tiny
    dw, db = (gp * n).sum(0), gp.sum(0)
    bw = rows * U * (gp * n).abs().sum(0) + (gp.abs() * dn).sum(0) + (dgp * n.abs()).sum(0) + we * dw.abs() + wtiny
    bb = rows * U * gp.abs().sum(0) + dgp.sum(0) + we * db.abs() + wtiny
    return [1.01 * t for t in (by, bx, bw, bb)]


def _compare(got, want, bounds):
    names = ("y", "dx", "dw", "db")
    for name, a, r, t in zip(names, got, want, bounds):
        a = a.detach().cpu().double()
        assert a.shape == r.shape, name
        err = (a - r).abs()
        bad = ~(err <= t)
        assert not bool(bad.any()), f"{name}: {int(bad.sum())} of {bad.numel()} beyond the bound, worst ratio {float((err / t).max()):.3f}"


def _state(dev, seed=1234567890123, offset=17):
    return torch.tensor([nd._signed(seed), nd._signed(offset)], dtype=torch.int64, device=dev)


def _run(x, act, w, b, normalize, p, state, go, eps=1e-5, sequence=0):
    leaves = [t.clone().requires_grad_() for t in (x, w, b)] if normalize else [x.clone().requires_grad_()]
    y = nd.activate_norm_dropout(leaves[0], act, *(leaves[1:] if normalize else (None, None)), normalize=normalize, eps=eps, p=p,
                                 state=state, sequence=sequence)
    return (y,) + torch.autograd.grad(y, leaves, go)


SHAPES = [(1, 1), (5, 1), (1, 2), (3, 5), (7, 8), (2, 31), (9, 32), (70, 33), (13, 37), (600, 64), (33, 100), (131, 128), (65, 255),
          (64, 256), (40, 257), (21, 512), (30, 777), (5, 1000), (17, 1023), (19, 1024), (6, 1025), (9, 2048), (7, 2050), (3, 4099),
          (4, 8192), (2, 16385), (3, 40003)]


@pytest.mark.parametrize("types", ["fp32-fp32", "bf16-bf16", "bf16-fp32", "fp16-fp16", "fp16-fp32"])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: f"{s[0]}x{s[1]}")
def test_layer_norm_forward_backward(gpu_device, shape, types):
    dtype, wdtype = (DTYPES[t] for t in types.split("-"))
    x, w, b, go = _data(*shape, dtype, wdtype, seed=shape[1])
    xd, wd, bd = (t.to(gpu_device).requires_grad_() for t in (x, w, b))
    y = nd.layer_norm(xd, wd, bd, eps=1e-5)
    got = (y,) + torch.autograd.grad(y, (xd, wd, bd), go.to(gpu_device))
    assert [t.dtype for t in got] == [dtype, dtype, wdtype, wdtype]
    _compare(got, orc.tail(x, None, w, b, grad=go), _bounds(x, None, w, b, True, 1e-5, None, 0.0, go, dtype, wdtype))
    with torch.no_grad():
        assert torch.equal(nd.layer_norm(xd, wd, bd, eps=1e-5), y)  # inference: the same bits


@pytest.mark.parametrize("normalize", [True, False])
@pytest.mark.parametrize("act", [None] + ACTS)
@pytest.mark.parametrize("shape, types, p", [((37, 64), "fp32-fp32", 0.1), ((11, 333), "fp16-fp32", 0.3), ((5, 1030), "bf16-bf16", 0.0),
                                             ((9, 17), "bf16-fp32", 0.5), ((3, 4100), "fp32-fp32", 0.7), ((2, 16390), "fp32-fp32", 0.2)],
                         ids=lambda v: "x".join(map(str, v)) if isinstance(v, tuple) else str(v))
def test_activate_norm_dropout(gpu_device, shape, types, p, act, normalize):
    dtype, wdtype = (DTYPES[t] for t in types.split("-"))
    x, w, b, go = _data(*shape, dtype, wdtype, seed=shape[1] + 1)
    kept = orc.keep(x.numel(), p, 1234567890123, 17 + 3).view(shape) if p > 0 else None
    d = [t.to(gpu_device) for t in (x, w, b, go)]
    if act is None and not normalize and p == 0.0:
        assert nd.activate_norm_dropout(d[0], None, normalize=False) is d[0]  # nothing to do
        return
    got = _run(d[0], act, d[1], d[2], normalize, p, _state(gpu_device), d[3], sequence=3)
    args = (act, w, b) if normalize else (act, None, None)
    _compare(got, orc.tail(x, *args, normalize=normalize, kept=kept, p=p, grad=go),
             _bounds(x, act, w, b, normalize, 1e-5, kept, p, go, dtype, wdtype))
    if kept is not None:
        assert bool((got[0].cpu()[~kept] == 0).all())
    again = _run(d[0], act, d[1], d[2], normalize, p, _state(gpu_device), d[3], sequence=3)
    assert all(torch.equal(a, b) for a, b in zip(got, again))  # equal calls, equal bits


@pytest.mark.parametrize("rows, width", [(20736, 64), (5000, 128), (3001, 333), (4000, 1024), (999, 2051)])
def test_many_rows(gpu_device, rows, width):
    """More rows than one sweep of the grid takes: gradients of the weights join many partial sums."""
    x, w, b, go = _data(rows, width, torch.float32, torch.float32, seed=rows)
    kept = orc.keep(x.numel(), 0.1, 1234567890123, 17).view(x.shape)
    d = [t.to(gpu_device) for t in (x, w, b, go)]
    got = _run(d[0], "leakyrelu", d[1], d[2], True, 0.1, _state(gpu_device), d[3])
    _compare(got, orc.tail(x, "leakyrelu", w, b, kept=kept, p=0.1, grad=go),
             _bounds(x, "leakyrelu", w, b, True, 1e-5, kept, 0.1, go, torch.float32, torch.float32))


@pytest.mark.parametrize("n", [1, 2, 3, 4, 5, 63, 64, 255, 1000, 4097, 144002])
@pytest.mark.parametrize("p", [1e-12, 0.1, 0.5, 0.999, 1.0])
def test_keep_mask_and_dropout_match_the_oracle(gpu_device, n, p):
    seed, offset = (1 << 64) - 12345, (1 << 64) - 2  # offset + sequence passes 64 bits
    for sequence in (0, 3):
        state = _state(gpu_device, seed, offset)
        want = orc.keep(n, p, seed, offset + sequence)
        mask = nd.keep_mask(n, p, state, sequence)
        assert mask.dtype == torch.bool and torch.equal(mask.cpu(), want)
        for dtype in DTYPES.values():
            x = torch.randn(n, generator=torch.Generator().manual_seed(n)).to(dtype)
            xd = x.to(gpu_device).requires_grad_()
            y = nd.dropout(xd, p, state, sequence=sequence)
            g, = torch.autograd.grad(y, xd, xd.detach())
            scale = torch.tensor(1.0 / (1.0 - p) if p < 1 else 0.0, dtype=torch.float32)
            ref = torch.where(want, x.float() * scale, torch.zeros(n)).to(dtype)  # one product, one rounding: equal bits
            assert torch.equal(y.detach().cpu(), ref) and torch.equal(g.cpu(), ref)


def test_mask_does_not_depend_on_shape_type_or_operator(gpu_device):
    state = _state(gpu_device)
    mask = nd.keep_mask(6 * 10 * 35, 0.4, state)
    for shape in ((2100,), (2100, 1), (60, 35), (6, 10, 35), (1, 2100), (35, 60)):
        for dtype in DTYPES.values():
            one = torch.ones(shape, dtype=dtype, device=gpu_device)
            assert torch.equal(nd.dropout(one, 0.4, state) != 0, mask.view(shape))
            y = nd.activate_norm_dropout(one, "relu", None, torch.ones(shape[-1], device=gpu_device), p=0.4, state=state)
            assert torch.equal(y != 0, mask.view(shape))


def test_dropped_places_hold_zero_whatever_they_held(gpu_device):
    state = _state(gpu_device)
    for dtype in DTYPES.values():
        for bad in (float("nan"), float("inf"), float("-inf")):
            x = torch.full((37, 29), bad, dtype=dtype, device=gpu_device, requires_grad=True)
            keep = nd.keep_mask(x.numel(), 0.5, state).view(x.shape)
            for act in (None, "relu", "gelu"):
                y = nd.activate_norm_dropout(x, act, normalize=False, p=0.5, state=state)
                assert bool((y[~keep] == 0).all()) and not bool(torch.signbit(y[~keep]).any())
            y = nd.dropout(x, 0.5, state)
            assert bool((~torch.isfinite(y[keep])).all())
            g, = torch.autograd.grad(y, x, torch.full_like(x, bad))
            assert bool((g[~keep] == 0).all()) and bool((~torch.isfinite(g[keep])).all())
    # one bad value makes its own row NaN and no other
    x = torch.randn(9, 64, device=gpu_device)
    x[4, 7] = float("inf")
    y = nd.layer_norm(x)
    assert bool(torch.isnan(y[4]).all()) and bool(torch.isfinite(y[[0, 1, 2, 3, 5, 6, 7, 8]]).all())


@pytest.mark.parametrize("act", ACTS)
def test_activations_over_the_whole_range(gpu_device, act):
    """Alone, in fp32, from -1e30 to 1e30 and NaN: value and derivative against float64.  The docstring's bounds (4 u |x| + 4 u |a|,
    8 u (1 + |x|)) up to |x| = 90; beyond that every activation is 0, -1, 1 or x and its derivative 0 or 1."""
    g = torch.Generator().manual_seed(6)
    x = torch.cat([torch.linspace(-90, 90, 20001), torch.randn(20000, generator=g), torch.randn(20000, generator=g) * 1e-3,
                   torch.tensor([0.0, -0.0, 1e-30, -1e-30, 1e-40, -1e-40, 0.5, -0.5, 20.0, 20.5, -20.0, 200.0, -200.0, 1e30, -1e30])])
    xd = x.to(gpu_device).requires_grad_()
    y = nd.activate_norm_dropout(xd, act, normalize=False)
    dy, = torch.autograd.grad(y, xd, torch.ones_like(xd))
    xr = x.double().requires_grad_()
    want = orc.act(xr, act)
    dwant, = torch.autograd.grad(want.sum(), xr)
    far = xr.detach().abs().clamp(max=90)  # beyond: the value itself is exact, errors do not grow
    err, derr = (y.detach().cpu().double() - want.detach()).abs(), (dy.cpu().double() - dwant).abs()
    assert bool((err <= 4 * U * far + 5 * U * want.detach().abs() + 1e-37).all()), float((err / (far + 1e-30)).max() / U)
    assert bool((derr <= 8 * U * (1 + far)).all()), float((derr / (1 + far)).max() / U)
    odd = torch.tensor([float("nan"), float("inf")], device=gpu_device, requires_grad=True)
    got = nd.activate_norm_dropout(odd, act, normalize=False)
    grad, = torch.autograd.grad(got, odd, torch.ones_like(odd))
    assert act in ("relu", "leakyrelu") or bool(torch.isnan(grad[0]))  # those two: a comparison, as torch's
    assert bool(torch.isnan(got[0])) and float(got[1].detach()) == (1.0 if act == "tanh" else float("inf"))


def test_constant_and_extreme_rows(gpu_device):
    w, b = torch.rand(100, device=gpu_device) + 0.5, torch.rand(100, device=gpu_device)
    for value in (0.0, 1.0, -3.75, 2.0 ** 60):  # sums of 100 equal powers-of-two multiples are exact: variance 0, y = bias
        assert torch.equal(nd.layer_norm(torch.full((3, 100), value, device=gpu_device), w, b), b.expand(3, 100))
    assert bool(torch.isnan(nd.layer_norm(torch.zeros(2, 8, device=gpu_device), eps=0.0)).all())  # 0 / 0, as torch
    # no eps and a variance far below the smallest normal number, or one that overflows (1 / sqrt(inf) = 0: the bias alone)
    x = torch.randn(7, 100, generator=torch.Generator().manual_seed(3))
    want = orc.tail(x, eps=0.0)[0]
    for scale in (2.0 ** -66, 2.0 ** -50, 1.0, 2.0 ** 50):
        got = nd.layer_norm((x * scale).to(gpu_device), eps=0.0).cpu().double()
        # below 2^-126 the variance itself has fewer bits: 2^-132 keeps 17 of them, half of that relative error reaches y
        assert float((got - want).abs().max()) <= (64 * U if scale > 2.0 ** -60 else 2.0 ** -16) * float(want.abs().max()), scale
    assert torch.equal(nd.layer_norm((x * 1e25).to(gpu_device), w, b), b.expand(7, 100))
    # a large common offset: the variance is formed from differences, not from squares.  Offset 4096 + k / 4 is exact in fp32,
    # the mean of 64 such values too
    x = 4096.0 + torch.arange(64.0).repeat(5, 1) / 4
    got = nd.layer_norm(x.to(gpu_device)).cpu().double()
    want = orc.tail(x)[0]
    assert float((got - want).abs().max()) <= 16 * U * float(want.abs().max())


def test_affine_parts_may_be_absent_or_frozen(gpu_device):
    x, w, b, go = _data(50, 96, torch.float32, torch.float32, seed=5)
    d = [t.to(gpu_device) for t in (x, w, b, go)]
    xr, wr, br = (t.clone().requires_grad_() for t in d[:3])
    full = torch.autograd.grad(nd.layer_norm(xr, wr, br), (xr, wr, br), d[3])
    # any subset of the leaves: the same bits
    for names in ("x", "w", "b", "xw", "xb", "wb"):
        leaves = {k: t.clone().requires_grad_(k in names) for k, t in zip("xwb", d[:3])}
        y = nd.layer_norm(leaves["x"], leaves["w"], leaves["b"])
        for k, g in zip(names, torch.autograd.grad(y, [leaves[k] for k in names], d[3])):
            assert torch.equal(g, full["xwb".index(k)]), (names, k)
    ones, zeros = torch.ones_like(d[1]), torch.zeros_like(d[2])
    for weight, bias in ((None, None), (d[1], None), (None, d[2])):
        x1, x2 = (d[0].clone().requires_grad_() for _ in range(2))
        y1 = nd.layer_norm(x1, weight, bias)
        y2 = nd.layer_norm(x2, ones if weight is None else weight, zeros if bias is None else bias)
        assert torch.equal(y1, y2)
        assert torch.equal(*(torch.autograd.grad(y, t, d[3])[0] for y, t in ((y1, x1), (y2, x2))))


def test_strides_orders_and_misaligned_rows(gpu_device):
    state = _state(gpu_device)
    base = torch.randn(66, 140, device=gpu_device)
    w, b = torch.randn(64, device=gpu_device), torch.randn(64, device=gpu_device)
    wide = torch.randn(200, device=gpu_device)
    views = [base[:, :64], base[:, 1:65], base[:, 3:67], base[::3, 5:69], base.view(3, 22, 140)[:, :, 7:71], base[:1, 2:66].expand(9, 64),
             base[:, :128:2], base[:64, :64].t(), base.view(3, 22, 140).transpose(0, 1)[:, :, :64], base[4, 9:73], base[:0, :64]]
    for dtype in DTYPES.values():
        for v in views:
            v = v.to(dtype) if dtype != torch.float32 else v
            if dtype != torch.float32 and v.dim() == 2 and v.shape[0] > 1:  # keep a row stride after the conversion
                v = torch.cat([v, v], 1)[:, 1:65]
            dense = v.clone(memory_format=torch.contiguous_format)
            g = torch.randn(v.shape[:-1] + (80,), device=gpu_device).to(dtype)[..., 3:67]
            res = []
            for x, go in ((v, g), (dense, g.contiguous()), (v, g.flip(-1).flip(-1))):
                x, wr, br = x.detach().requires_grad_(), w.clone().requires_grad_(), b.clone().requires_grad_()
                out = nd.activate_norm_dropout(x, "tanh", wr, br, p=0.2, state=state)
                plain = nd.activate_norm_dropout(x, "silu", normalize=False, p=0.2, state=state)
                assert out.is_contiguous() and out.shape == v.shape
                res.append((out, plain) + torch.autograd.grad(out, (x, wr, br), go) + torch.autograd.grad(plain, x, go))
            for other in res[1:]:
                assert all(torch.equal(a, c) for a, c in zip(res[0], other))
    # a gradient expanded from one value, as y.sum() hands it over; weights that are views
    x = base[:, :64].detach().requires_grad_()
    wv = wide[::3][:64].detach().requires_grad_()
    nd.layer_norm(x, wv, wide[5:69]).sum().backward()
    x2, w2 = base[:, :64].contiguous().requires_grad_(), wv.detach().contiguous().requires_grad_()
    nd.layer_norm(x2, w2, wide[5:69].contiguous()).backward(torch.ones(66, 64, device=gpu_device))
    assert torch.equal(x.grad, x2.grad) and torch.equal(wv.grad, w2.grad)


def test_neighbours_of_the_outputs_stay(gpu_device):
    """C entry: rows of y, statistics and gradients inside larger buffers; nothing before or behind them is written."""
    import ctypes as C

    from amber_amd import _lib
    lib = _lib.load()
    stream = _lib.stream_ptr(gpu_device)
    for dtype, rows, width in ((torch.float32, 5, 67), (torch.bfloat16, 3, 1031), (torch.float16, 70, 40), (torch.float32, 2, 17001)):
        n = rows * width
        x, w, b, go = (t.to(gpu_device) for t in _data(rows, width, dtype, dtype, seed=3))
        name = _lib.DTYPE[str(dtype).split(".")[1]]
        desc = C.byref(_lib.AmberTailDesc(dtype=name, weight_dtype=name, activation=1, normalize=1, p=0.3,
                                          eps=1e-5, sequence=0))
        state = _state(gpu_device)
        bufs = [torch.full((k + 128,), 7.0, dtype=t, device=gpu_device)
                for k, t in ((n, dtype), (2 * rows, torch.float32), (n, dtype), (width, dtype), (width, dtype))]
        y, stats, gx, gw, gb = (t.data_ptr() + 64 * t.element_size() for t in bufs)
        assert lib.amber_mpn_tail_forward(desc, rows, width, x.data_ptr(), width, w.data_ptr(), b.data_ptr(), state.data_ptr(), y, stats,
                                          stream) == 0
        need = lib.amber_mpn_tail_backward_workspace_bytes(desc, rows, width)
        ws = torch.full((need + 256,), 9, dtype=torch.uint8, device=gpu_device)
        assert lib.amber_mpn_tail_backward(desc, rows, width, x.data_ptr(), width, go.data_ptr(), width, w.data_ptr(), stats,
                                           state.data_ptr(), gx, gw, gb, ws.data_ptr(), need, stream) == 0
        for t in bufs:
            assert bool((t[:64] == 7).all()) and bool((t[-64:] == 7).all()) and bool((t[64:-64] != 7).all())
        assert bool((ws[need:] == 9).all())


def test_empty_batches(gpu_device):
    state = _state(gpu_device)
    x = torch.randn(0, 48, device=gpu_device, requires_grad=True)
    w, b = (torch.randn(48, device=gpu_device, requires_grad=True) for _ in range(2))
    y = nd.activate_norm_dropout(x, "relu", w, b, p=0.5, state=state)
    gx, gw, gb = torch.autograd.grad(y, (x, w, b), torch.randn(0, 48, device=gpu_device))
    assert y.shape == gx.shape == (0, 48) and not bool(gw.any()) and not bool(gb.any())
    z = torch.randn(5, 0, device=gpu_device, requires_grad=True)
    d = nd.dropout(z, 0.5, state)
    assert d.shape == (5, 0) and torch.autograd.grad(d, z, torch.empty(5, 0, device=gpu_device))[0].shape == (5, 0)
    assert nd.keep_mask(0, 0.5, state).shape == (0,)
    s = torch.tensor(3.0, device=gpu_device, requires_grad=True)  # no dimensions: one element
    assert nd.dropout(s, 1.0, state).shape == () and float(nd.dropout(s, 1.0, state).detach()) == 0.0


def test_identities(gpu_device):
    x = torch.randn(4, 8, device=gpu_device)
    assert nd.dropout(x, 0.0) is x and nd.dropout(x, 0.7, training=False) is x
    assert nd.activate_norm_dropout(x, None, normalize=False, p=0.5, training=False) is x
    assert torch.equal(nd.activate_norm_dropout(x, "relu", p=0.5, training=False), nd.activate_norm_dropout(x, "relu"))


def test_refusals(gpu_device):
    x = torch.randn(4, 8, device=gpu_device)
    state = _state(gpu_device)
    with pytest.raises(TypeError, match="float32, bfloat16 or float16"):
        nd.layer_norm(x.double())
    with pytest.raises(ValueError, match="needs the generator"):
        nd.dropout(x, 0.5)
    with pytest.raises(ValueError, match="the data on"):
        nd.dropout(x, 0.5, state.cpu())
    with pytest.raises(ValueError, match="contiguous int64"):
        nd.activate_norm_dropout(x, "relu", p=0.5, state=state.float())
    with pytest.raises(ValueError, match="Unknown activation"):
        nd.activate_norm_dropout(x, "swiglu")
    with pytest.raises(ValueError, match="without normalize"):
        nd.activate_norm_dropout(x, "relu", x[0], normalize=False)
    with pytest.raises(ValueError, match="is on"):
        nd.layer_norm(x, torch.ones(8))
    with pytest.raises(ValueError, match="weight of shape"):
        nd.layer_norm(x, torch.ones(7, device=gpu_device))
    xr = x.clone().requires_grad_()
    g, = torch.autograd.grad(nd.layer_norm(xr).pow(2).sum(), xr, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()  # first derivatives only
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y = nd.dropout(xr, 0.5, state)
        state.add_(1)  # the backward pass would draw other numbers
        y.sum().backward()
    for view in (lambda t: t, lambda t: t[:, 1:]):  # the input as well, read in place or not
        base = xr * 2
        y = nd.layer_norm(view(base))
        base.add_(1)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            y.sum().backward()
    y = nd.layer_norm(xr)
    y.sum().backward()
    with pytest.raises(RuntimeError, match="second time"):
        y.sum().backward()


def test_gradients_against_differences(gpu_device):
    """Central differences along random directions: truncation h^2 / 6 of the third derivative and rounding u |f| / h; with h = 2^-6 and
    f a sum of 40 x 24 terms of order 1 both are below 1 % of the directional derivative's scale |grad| |dir|."""
    state = _state(gpu_device)
    gen = torch.Generator().manual_seed(2)
    x, w, b, go = _data(40, 24, torch.float32, torch.float32, seed=8)
    d = [t.to(gpu_device) for t in (x, w, b, go)]
    for act in (None, "tanh", "silu", "mish", "gelu"):
        grads = _run(d[0], act, d[1], d[2], True, 0.25, state, d[3])[1:]
        f = lambda *t: float((nd.activate_norm_dropout(t[0], act, t[1], t[2], p=0.25, state=state).double() * d[3].double()).sum())  # noqa: E731
        for k in range(3):
            v = torch.randn(d[k].shape, generator=gen).to(gpu_device)
            v = v / v.norm()
            h = 2.0 ** -6
            lo, hi = ([t + s * h * v if i == k else t for i, t in enumerate(d[:3])] for s in (-1, 1))
            diff = (f(*hi) - f(*lo)) / (2 * h)
            assert abs(diff - float((grads[k].double() * v.double()).sum())) <= 0.01 * float(grads[k].double().norm()), (act, k)


def test_zero_and_negated_tensors(gpu_device):
    """Tensors whose memory does not hold their values: a negated view, a gradient of zeros without memory."""
    x = torch.randn(6, 40, dtype=torch.complex64, device=gpu_device).conj().imag
    assert x.is_neg()
    assert torch.equal(nd.layer_norm(x), nd.layer_norm(x.clone())) and torch.equal(nd.dropout(x, 0.3, _state(gpu_device)),
                                                                                   nd.dropout(x.clone(), 0.3, _state(gpu_device)))
    xr, w = torch.randn(6, 40, device=gpu_device, requires_grad=True), torch.randn(40, device=gpu_device, requires_grad=True)
    zero = torch._efficientzerotensor((6, 40), device=gpu_device)
    gx, gw = torch.autograd.grad(nd.layer_norm(xr, w), (xr, w), zero)
    assert not bool(gx.any()) and not bool(gw.any())
    y = nd.layer_norm(xr, w)
    g = torch.randn(6, 40, dtype=torch.complex64, device=gpu_device).conj().imag
    a = torch.autograd.grad(y, (xr, w), g, retain_graph=True)
    assert all(torch.equal(s, t) for s, t in zip(a, torch.autograd.grad(y, (xr, w), g.clone())))  # and twice through one graph


def test_generator_buffer_as_state_is_guarded(gpu_device):
    gen = nd.CounterGenerator(3, device=gpu_device)
    x = torch.randn(5, 5, device=gpu_device, requires_grad=True)
    y = nd.dropout(x, 0.5, gen.state)
    gen.take()  # moves the offset that the backward pass would read
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


@pytest.mark.parametrize("shape", [(60, 64), (5, 12, 64)])
def test_saved_tensors_may_move(gpu_device, shape):
    """x, weight, statistics and state go through the host and come back contiguous, whatever rows x had in the forward pass; x alone
    comes back with rows further apart; a hook that changes the type is refused."""
    base = torch.randn(*shape[:-1], 130, device=gpu_device)
    w, b = torch.randn(64, device=gpu_device), torch.randn(64, device=gpu_device)
    state, go = nd.CounterGenerator(3, gpu_device).take(), torch.randn(shape, device=gpu_device)

    def gradients(x, hooks):
        leaves = [t.detach().clone().requires_grad_() for t in (w, b)]
        xl = x.detach().requires_grad_()
        with hooks:
            y = nd.activate_norm_dropout(xl, "silu", *leaves, p=0.25, state=state)
            z = nd.activate_norm_dropout(y, "mish", normalize=False, p=0.25, state=state, sequence=1)
        return torch.autograd.grad(z, [xl, *leaves], go)

    def keep(t):
        return t

    def spread(t):
        if t.dim() < 2:
            return t
        wide = t.new_full((*t.shape[:-1], t.shape[-1] + 7), float("nan"))
        wide[..., :t.shape[-1]] = t
        return wide[..., :t.shape[-1]]

    for x in (base[..., :64], base[..., 3:67], base[..., :64].contiguous()):
        want = gradients(x, torch.autograd.graph.saved_tensors_hooks(keep, keep))
        for hooks in (torch.autograd.graph.save_on_cpu(), torch.autograd.graph.saved_tensors_hooks(keep, spread)):
            for a, b_ in zip(want, gradients(x, hooks)):
                assert torch.equal(a, b_)
    with pytest.raises(RuntimeError, match="came back as another tensor"):
        gradients(base[..., :64], torch.autograd.graph.saved_tensors_hooks(keep, lambda t: t.double()))


def test_recomputed_layers(gpu_device):
    """torch.utils.checkpoint with the range taken outside gives the gradients of the plain call."""
    x, state = torch.randn(50, 70, device=gpu_device), nd.CounterGenerator(4, gpu_device).take()
    w = torch.randn(70, device=gpu_device, requires_grad=True)
    want = None
    for reentrant in (None, False, True):
        xl = x.clone().requires_grad_()
        f = lambda t: nd.activate_norm_dropout(t * 2, "elu", w, p=0.3, state=state)
        y = f(xl) if reentrant is None else torch.utils.checkpoint.checkpoint(f, xl, use_reentrant=reentrant)
        w.grad = None
        y.square().sum().backward()
        got = (y.detach(), xl.grad, w.grad)
        want = want or got
        assert all(torch.equal(a, b) for a, b in zip(want, got))


def test_inference_mode(gpu_device):
    x = torch.randn(9, 33, device=gpu_device)
    with torch.inference_mode():
        gen = nd.CounterGenerator(8, gpu_device)
        a = nd.activate_norm_dropout(x, "relu", p=0.5, state=gen.take())
    outside = nd.CounterGenerator(8, gpu_device)
    assert torch.equal(a, nd.activate_norm_dropout(x, "relu", p=0.5, state=outside.take()))
    with torch.inference_mode():
        gen.take(), outside.take()
        assert gen.get_state() == outside.get_state() == (8, 2)


def test_forward_mode_is_refused(gpu_device):
    import torch.autograd.forward_ad as fwd
    x = torch.randn(4, 8, device=gpu_device)
    with fwd.dual_level():
        with pytest.raises(NotImplementedError, match="forward-mode"):
            nd.layer_norm(fwd.make_dual(x, torch.ones_like(x)))


def test_one_dimension_beyond_32_bits(gpu_device):
    n = (1 << 32) + 7
    x = torch.ones(n, dtype=torch.bfloat16, device=gpu_device)
    y = nd.dropout(x, 0.5, _state(gpu_device))
    assert torch.equal(y[-11:].cpu(), orc.keep(11, 0.5, 1234567890123, 17, start=n - 11).to(torch.bfloat16) * 2)


def test_offsets_beyond_32_bits(gpu_device):
    """More than 2^32 elements in 16 bits (8.6 GB a tensor): the last rows are right, forward and backward."""
    rows, width = (1 << 32) // 4096 + 5, 4096
    state = _state(gpu_device)
    x = torch.zeros(rows, width, dtype=torch.bfloat16, device=gpu_device)
    last = 3
    tail, w, b, go = _data(last, width, torch.bfloat16, torch.bfloat16, seed=4)
    x[-last:] = tail.to(gpu_device)
    kept = orc.keep(last * width, 0.3, 1234567890123, 17, start=(rows - last) * width).view(last, width)
    y = nd.dropout(x, 0.3, state)
    scale = torch.tensor(1.0 / 0.7, dtype=torch.float32)
    assert torch.equal(y[-last:].cpu(), torch.where(kept, tail.float() * scale, torch.zeros(())).to(torch.bfloat16))
    del y
    xr, wr, br = x.requires_grad_(), w.to(gpu_device).requires_grad_(), b.to(gpu_device).requires_grad_()
    y = nd.activate_norm_dropout(xr, "leakyrelu", wr, br, p=0.3, state=state)
    g = torch.zeros_like(x)
    g[-last:] = go.to(gpu_device)  # only these rows reach the gradients of the weights
    gx, gw, gb = torch.autograd.grad(y, (xr, wr, br), g)
    got = (y[-last:], gx[-last:], gw, gb)
    _compare(got, orc.tail(tail, "leakyrelu", w, b, kept=kept, p=0.3, grad=go),
             _bounds(tail, "leakyrelu", w, b, True, 1e-5, kept, 0.3, go, torch.bfloat16, torch.bfloat16))
    assert not bool(gx[:-last].any())
    del y, gx, g
    mask = nd.keep_mask((1 << 32) + 9, 0.3, state)
    assert torch.equal(mask[-9:].cpu(), orc.keep(9, 0.3, 1234567890123, 17, start=1 << 32))


@pytest.mark.parametrize("megabytes", [150, 220, 330])
@pytest.mark.parametrize("width, dtype", [(128, "fp32"), (1021, "fp32"), (333, "fp16"), (4099, "bf16"), (16400, "bf16")])
def test_large_calls_give_the_small_calls_rows(gpu_device, width, dtype, megabytes):
    """Tensors around what the caches hold: every row of a large call has the bits of the same row in a call of a few rows, and the
    dropped places are the mask's."""
    t = DTYPES[dtype]
    rows = megabytes * 10 ** 6 // (width * t.itemsize) + 1
    torch.manual_seed(width + megabytes)
    x, g = (torch.randn(rows, width, device=gpu_device, dtype=t) for _ in range(2))
    w, b, state = torch.randn(width, device=gpu_device), torch.randn(width, device=gpu_device), _state(gpu_device)

    def both(x, g, **kw):
        xr = x.detach().requires_grad_()
        y = nd.activate_norm_dropout(xr, "leakyrelu", **kw)
        return y.detach(), torch.autograd.grad(y, xr, g)[0]

    for kw in (dict(weight=w, bias=b), dict(normalize=False)):
        large = both(x, g, **kw)
        for first in (0, rows // 2, rows - 7):
            small = both(x[first:first + 7], g[first:first + 7], **kw)
            assert all(torch.equal(a[first:first + 7], c) for a, c in zip(large, small))
        for part in torch.arange(rows, device=gpu_device).split(rows // 9 + 1):  # all rows, a ninth at a time
            small = both(x[part[0]:part[-1] + 1], g[part[0]:part[-1] + 1], **kw)
            assert all(torch.equal(a[part[0]:part[-1] + 1], c) for a, c in zip(large, small))
    keep = nd.keep_mask(x.numel(), 0.25, state).view(x.shape)
    y, dx = both(x, g, normalize=False, p=0.25, state=state)
    scale = torch.tensor(1 / 0.75, dtype=torch.float32, device=gpu_device)
    slope = torch.where(x > 0, 1.0, torch.tensor(0.01, device=gpu_device))
    assert torch.equal(y, torch.where(keep, x.float() * slope * scale, 0.0).to(t))
    assert torch.equal(dx, torch.where(keep, g.float() * scale * slope, 0.0).to(t))


def test_other_stream_and_two_at_once(gpu_device):
    x, w, b, go = (t.to(gpu_device) for t in _data(3000, 200, torch.float32, torch.float32, seed=9))
    state = _state(gpu_device)
    want = _run(x, "gelu", w, b, True, 0.1, state, go)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for s in streams:
        with torch.cuda.stream(s):
            got.append(_run(x, "gelu", w, b, True, 0.1, state, go))
    torch.cuda.synchronize()
    for res in got:
        assert all(torch.equal(a, c) for a, c in zip(res, want))


def test_generator_ranges_are_disjoint(gpu_device):
    gen = nd.CounterGenerator(99, device=gpu_device)
    taken = [gen.take(k) for k in (1, 3, 2)]
    assert [t.tolist() for t in taken] == [[99, 0], [99, 1], [99, 4]] and gen.get_state() == (99, 6)
    gen.set_state(5, (1 << 64) - 1)
    assert gen.take(2).tolist() == [5, -1] and gen.get_state() == (5, 1)
    s = [torch.cuda.Stream() for _ in range(2)]
    offsets = []
    for i in range(6):
        with torch.cuda.stream(s[i % 2]):
            offsets.append(gen.take())
    torch.cuda.synchronize()
    assert sorted(t.tolist()[1] for t in offsets) == list(range(1, 7))


def test_captured_step_draws_anew_at_every_replay(gpu_device):
    """take, forward and backward in one graph: every replay equals the eager step at the generator's offset of that replay."""
    x, w, b, go = (t.to(gpu_device) for t in _data(500, 96, torch.float32, torch.float32, seed=12))
    gen = nd.CounterGenerator(4242, device=gpu_device)

    def step():
        state = gen.take(2)
        xr, wr, br = (t.detach().requires_grad_() for t in (x, w, b))
        h = nd.activate_norm_dropout(xr, "silu", wr, br, p=0.2, state=state)
        y = nd.dropout(h, 0.3, state, sequence=1)
        return (y.detach(),) + torch.autograd.grad(y, (xr, wr, br), go)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    seen = []
    for replay in range(4):
        gen.set_state(4242, 100 + 2 * replay)
        eager = step()
        gen.set_state(4242, 100 + 2 * replay)
        graph.replay()
        torch.cuda.synchronize()
        assert gen.get_state() == (4242, 102 + 2 * replay)
        assert all(torch.equal(a, c) for a, c in zip(out, eager))
        seen.append(out[0].clone())
    graph.replay()  # without resetting the generator: the next range
    torch.cuda.synchronize()
    assert gen.get_state() == (4242, 110)
    assert all(not torch.equal(out[0], t) for t in seen)


def test_two_graphs_of_one_generator(gpu_device):
    """Steps of two sizes, captured one by one from one generator and replayed in turn with eager steps between them: each draws the
    generator's next range, and neither disturbs the other's workspace."""
    gen, graphs = nd.CounterGenerator(77, device=gpu_device), []
    sizes = ((900, 96), (70, 1030))
    data = [tuple(t.to(gpu_device) for t in _data(*size, torch.float32, torch.float32, seed=13 + i)) for i, size in enumerate(sizes)]

    def step(x, w, b, go):
        state = gen.take()
        xr, wr, br = (t.detach().requires_grad_() for t in (x, w, b))
        y = nd.activate_norm_dropout(xr, "leakyrelu", wr, br, p=0.2, state=state)
        return (y.detach(),) + torch.autograd.grad(y, (xr, wr, br), go)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for d in data:
            step(*d)
    torch.cuda.current_stream().wait_stream(side)
    for d in data:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step(*d)
        graphs.append((graph, out))
    gen.set_state(77, 0)
    got = []
    for which in (0, 1, 1, 0, 2, 0, 1):  # 2: an eager step
        if which == 2:
            step(*data[0])
            got.append(None)
            continue
        graphs[which][0].replay()
        got.append((which, [t.clone() for t in graphs[which][1]]))
    torch.cuda.synchronize()
    assert gen.get_state() == (77, len(got))
    gen.set_state(77, 0)
    for entry in got:
        want = step(*data[entry[0] if entry else 0])
        assert entry is None or all(torch.equal(a, c) for a, c in zip(entry[1], want))


def _decoder(norm, p, act, layers=2, latent=64):
    return AttrDict({"activation_function": act, "num_layers": layers,
                     "regularization": {"dropout": p, "spectral_norm": False, "latent_normalization": norm}})


@pytest.mark.parametrize("norm, p, act", [("layer", 0.3, "leakyrelu"), (None, 0.3, "gelu"), ("layer", 0.0, "mish"), ("batch", 0.25, "elu")])
def test_decoder_layers_in_one_pass_each(gpu_device, norm, p, act):
    """MLP.run_layers with a generator against the same layers in float64 with the generator's masks: 2e-5 of each tensor's largest
    value (products of 64 terms twice in a row: a few u sqrt(64) each, with the norms' and batch statistics' amplification)."""
    torch.manual_seed(3)
    mlp = MLP(in_features=64, latent_dimension=64, mlp_config=_decoder(norm, p, act)).to(gpu_device).train()
    for k, q in mlp.named_parameters():
        with torch.no_grad():
            q.add_(0.1 * torch.randn_like(q))
    x = torch.randn(700, 64, device=gpu_device, requires_grad=True)
    go = torch.randn(700, 64, device=gpu_device)
    gen = nd.CounterGenerator(31, device=gpu_device)
    import copy
    ref = copy.deepcopy(mlp).cpu().double()
    y = mlp.run_layers(x, gen)
    grads = torch.autograd.grad(y, [x] + list(mlp.parameters()), go)
    assert gen.get_state() == (31, 2 if p else 0)
    xr = x.detach().cpu().double().requires_grad_()
    t, k = xr, 0
    for layer in ref.mlp_layers:
        if isinstance(layer, torch.nn.Dropout):
            kept = orc.keep(t.numel(), p, 31, k).view(t.shape)
            t = torch.where(kept, t / (1 - p), torch.zeros((), dtype=torch.float64))
            k += 1
        else:
            t = layer(t)
    want = torch.autograd.grad(t, [xr] + list(ref.parameters()), go.cpu().double())
    for a, r in zip((y.detach(),) + grads, (t.detach(),) + want):
        if act == "leakyrelu" and a.shape == x.shape and a is not y:
            continue  # a value within rounding of the kink takes the other slope
        assert float((a.cpu().double() - r).abs().max()) <= 2e-5 * float(r.abs().max()) + 1e-7
    if norm == "batch":
        for a, r in zip(mlp.buffers(), ref.buffers()):
            assert torch.allclose(a.cpu().double(), r.double(), rtol=1e-5, atol=1e-6)


def test_training_step_with_the_counter_generator(gpu_device):
    """The whole path: edge dropout and decoder dropout of a SupervisedMPN from one generator.  Equal states give equal outputs and
    gradients, other states others; the kept edges are the oracle's; inference is what it is without the generator."""
    g = syn.grid_batch(num_graphs=2, nx=9, ny=8, in_node_features=5, in_edge_features=2).to(gpu_device)
    cfg = default_architecture(latent_dimension=64, num_steps=2)
    cfg["decoder"] = _decoder("layer", 0.2, "leakyrelu")
    torch.manual_seed(5)
    plain = SupervisedMPN(cfg, g).to(gpu_device)
    model = SupervisedMPN(AttrDict(cfg, dropout_generator="counter", dropout_seed=7), g).to(gpu_device)
    model.load_state_dict(plain.state_dict(), strict=True)
    gen = model.mpn.dropout_generator
    assert gen.state.is_cuda
    edges = g.edge_index.shape[1]

    def step(offset):
        gen.set_state(7, offset)
        model.train().zero_grad(set_to_none=True)
        out = model(g)
        out.square().mean().backward()
        return [out.detach()] + [q.grad.clone() for q in model.parameters()]

    a, b, c = step(0), step(0), step(3)
    assert gen.get_state() == (7, 6)  # one range for the edges, two for the decoder
    assert all(torch.equal(s, t) for s, t in zip(a, b)) and not torch.equal(a[0], c[0])
    assert all(bool(torch.isfinite(t).all()) for t in a)
    work, csr = (gen.set_state(7, 50), model.mpn.prepare(g))[1]
    kept = orc.keep(edges, 0.1, 7, 50)
    assert torch.equal(work.edge_index.cpu(), g.edge_index.cpu()[:, kept]) and torch.equal(work.edge_attr.cpu(), g.edge_attr.cpu()[kept])
    with torch.no_grad():
        assert torch.equal(model.eval()(g), plain.eval()(g))


@pytest.mark.parametrize("width", [6, 33, 130, 257, 333, 515, 777, 1027, 2049, 4099, 8190, 9001])
def test_columns_held_twice_come_out_equal(gpu_device, width):
    """Odd widths: two lanes hold and store some columns.  Whoever stores last, the bits are the same: twenty runs, forward and back."""
    x, w, b, go = (t.to(gpu_device) for t in _data(400, width, torch.float32, torch.float32, seed=width))
    state = _state(gpu_device)
    first = _run(x, "tanh", w, b, True, 0.2, state, go)
    for _ in range(20):
        assert all(torch.equal(a, c) for a, c in zip(_run(x, "tanh", w, b, True, 0.2, state, go), first))


def test_run_to_run_equality_under_load(gpu_device):
    """Ten repetitions of a call that joins many partial sums: equal bits."""
    x, w, b, go = (t.to(gpu_device) for t in _data(30011, 128, torch.float32, torch.float32, seed=21))
    state = _state(gpu_device)
    first = _run(x, "elu", w, b, True, 0.15, state, go)
    for _ in range(10):
        assert all(torch.equal(a, c) for a, c in zip(_run(x, "elu", w, b, True, 0.15, state, go), first))
