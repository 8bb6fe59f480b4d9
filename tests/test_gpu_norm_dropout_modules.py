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


@pytest.mark.parametrize("width", [333, 1021, 1024, 4099, 8190, 16383, 40003, 999983])
@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_constant_rows_whose_sum_is_not_exact(gpu_device, width, dtype):
    """Rows of one value c: y is the bias and dx is 0 (up to the spread that the gradient alone has).  A first mean is off by some
    k u |c|, k <= 48 (a lane's elements or a compensated sum, then a tree); what the differences from it add up to takes that off again,
    to k u of it.  So |n| <= (48 u)^2 |c| / sqrt(eps), the statistics' mean is c to half a step, and n in the backward pass is at most
    u |c| / sqrt(eps)."""
    t, eps = DTYPES[dtype], 1e-5
    rows = 3
    gen = torch.Generator().manual_seed(width)
    w, b = 1 + 0.2 * torch.randn(width, generator=gen), 0.2 * torch.randn(width, generator=gen)
    go = torch.randn(rows, width, generator=gen).to(t)
    c = torch.tensor([[1000.1], [-0.3], [7.7]]).to(t)
    x = c.expand(rows, width).contiguous()
    got = _run(x.to(gpu_device), None, w.to(gpu_device), b.to(gpu_device), True, 0.0, None, go.to(gpu_device))
    cd, e = c.double().abs(), _half(t)[0]
    n = (48 * U) ** 2 * cd / math.sqrt(eps)
    y = got[0].cpu().double()
    assert bool(((y - b.double()).abs() <= 1.01 * (n * w.double().abs() + (2 * U + e) * b.double().abs())).all())
    # dx = rstd (h - mean h - n mean(h n)) with |n| <= u |c| / sqrt(eps)
    h = go.double() * w.double()
    r, nb = 1 / math.sqrt(eps), U * cd / math.sqrt(eps)
    want = r * (h - h.mean(1, keepdim=True))
    bound = r * (60 * U * (h.abs() + h.abs().mean(1, keepdim=True)) + nb * nb * h.abs().mean(1, keepdim=True)) + e * want.abs() + _half(t)[1]
    assert bool(((got[1].cpu().double() - want).abs() <= 1.01 * bound).all())


@pytest.mark.parametrize("rows, width", [(2, 16385), (3, 40003), (2, 999983), (1, 4194309)])
@pytest.mark.parametrize("offset", [0.0, 300.0])
def test_wide_rows_are_summed_as_accurately_as_narrow_ones(gpu_device, rows, width, offset):
    """The depth of a row held in registers whatever the width: forward with a mean far from 0, backward."""
    x, w, b, go = _data(rows, width, torch.float32, torch.float32, seed=width)
    x, go = x + offset, go + (0.5 if offset else 0.0)
    d = [t.to(gpu_device) for t in (x, w, b, go)]
    got = _run(d[0], None, d[1], d[2], True, 0.0, None, d[3])
    _compare(got, orc.tail(x, None, w, b, grad=go), _norm_bounds(x, w, b, go, chain=8))


@pytest.mark.parametrize("act, low, steps", [("silu", -60.0, 8), ("mish", -60.0, 13), ("gelu", -9.0, 18)])
def test_negative_tails_keep_their_relative_accuracy(gpu_device, act, low, steps):
    """fp32, relative to the value itself, which falls like exp(-|x|).  In u = 2^-24, the hardware's 2^x and reciprocal being within one
    unit in the last place (2 u): exp 4 (2^x, 1 + d, their product) and ln 2's own rounding, 1.9e-9 log2 e |x| = |x| / 20.  silu: 4 + 1
    (1 + e) + 2 (reciprocal) + 1.  mish: 4 x 4/3 (n = w (w + 2)) + 2 + 1 + 2 + 2, and 4/3 of ln 2's.  gelu: density 4, t 3 x 2.5 (how
    strongly t Q(t) depends on t), Horner's scheme 2.7, the fit 0.9, three products 3, ln 2's for x^2 / 2."""
    x = torch.linspace(low, -0.5, 200003)
    want = orc.act(x.double(), act)
    if act == "gelu":  # x Phi(x) by the complementary error function: 1 + erf(x) cancels
        want = 0.5 * x.double() * torch.erfc(-x.double() / math.sqrt(2.0))
    got = nd.activate_norm_dropout(x.to(gpu_device), act, normalize=False).cpu().double()
    power = x.double() ** 2 / 2 if act == "gelu" else x.double().abs() * (4 / 3 if act == "mish" else 1)
    worst = float((((got - want) / want).abs() / (U * (steps + power / 20))).max())
    assert worst <= 1.01, worst


def test_elu_derivative_keeps_its_relative_accuracy(gpu_device):
    """exp(x) within (4 + |x| / 20) u of itself (above)."""
    x = torch.linspace(-60.0, -1e-3, 200003)
    xd = x.to(gpu_device).requires_grad_()
    g, = torch.autograd.grad(nd.activate_norm_dropout(xd, "elu", normalize=False), xd, torch.ones_like(xd))
    assert float(((g.cpu().double() / x.double().exp() - 1).abs() / (4 + x.double().abs() / 20)).max()) <= 1.01 * U


@pytest.mark.parametrize("change", ["slope", "alpha", "approximate", "swapped", "act_hook", "norm_hook", "norm_pre_hook", "act_forward",
                                    "no_affine", "idle_dropout_hook"])
def test_decoder_layers_follow_their_modules(gpu_device, change):
    """run_layers with a generator computes what the modules in the list stand for at the call: parameters changed or modules exchanged
    after construction, hooks, a forward of their own.  Against the modules one by one in float64, with the generator's masks."""
    import copy
    nn = torch.nn
    act = {"slope": "leakyrelu", "alpha": "elu", "approximate": "gelu"}.get(change, "tanh")
    torch.manual_seed(8)
    mlp = MLP(in_features=64, latent_dimension=64, mlp_config=_decoder("layer", 0.25, act)).to(gpu_device).train()
    seen, mods = [], mlp.mlp_layers  # Linear, activation, LayerNorm, Dropout, twice
    if change == "slope":
        mods[1].negative_slope = 0.4
    elif change == "alpha":
        mods[5].alpha = 0.5
    elif change == "approximate":
        mods[1].approximate = "tanh"
    elif change == "swapped":
        mods[5] = nn.Softplus()
    elif change == "no_affine":
        mods[2] = nn.LayerNorm(64, elementwise_affine=False, eps=1e-2)
    elif change == "act_forward":
        mods[1].forward = lambda t: t * 2
    ref = copy.deepcopy(mlp).cpu().double()
    for m in (mods, ref.mlp_layers):
        if change == "act_hook":
            m[1].register_forward_hook(lambda mod, args, out: (seen.append(1), out * 3)[1])
        elif change == "norm_hook":
            m[2].register_forward_hook(lambda mod, args, out: (seen.append(1), out * 3)[1])
        elif change == "norm_pre_hook":
            m[6].register_forward_pre_hook(lambda mod, args: (seen.append(1), args[0] * args[0])[1])
        elif change == "idle_dropout_hook":  # not drawing: runs as the module it is
            m[3].p = 0.0
            m[3].register_forward_hook(lambda mod, args, out: (seen.append(1), out * 3)[1])
    x, go = torch.randn(200, 64), torch.randn(200, 64)
    xd = x.to(gpu_device).requires_grad_()
    gen = nd.CounterGenerator(3, device=gpu_device)
    y = mlp.run_layers(xd, gen)
    assert len(seen) == ("hook" in change)
    params = [q for q in mlp.parameters()]
    grads = torch.autograd.grad(y, [xd] + params, go.to(gpu_device))
    t = xr = x.double().requires_grad_()
    k = 0
    for layer in ref.mlp_layers:
        if isinstance(layer, nn.Dropout) and layer.p > 0:
            t = torch.where(orc.keep(t.numel(), 0.25, 3, k).view(t.shape), t / 0.75, torch.zeros((), dtype=torch.float64))
            k += 1
        else:
            t = layer(t)
    want = torch.autograd.grad(t, [xr] + list(ref.parameters()), go.double())
    assert gen.get_state() == (3, k)
    for name, a, r in zip(["y", "dx"] + [n for n, _ in mlp.named_parameters()], (y.detach(),) + grads, (t.detach(),) + want):
        if change == "slope" and name == "dx":
            continue  # a value within rounding of the kink takes the other slope
        assert float((a.cpu().double() - r).abs().max()) <= 2e-5 * float(r.abs().max()) + 1e-7, name


def test_hooks_on_a_drawing_dropout_are_refused(gpu_device):
    """The module itself would draw from torch's generator."""
    mlp = MLP(in_features=64, latent_dimension=64, mlp_config=_decoder("layer", 0.25, "tanh")).to(gpu_device).train()
    gen = nd.CounterGenerator(3, device=gpu_device)
    handle = mlp.mlp_layers[7].register_forward_hook(lambda mod, args, out: out)
    with pytest.raises(RuntimeError, match="dropout_generator"):
        mlp.run_layers(torch.randn(5, 64, device=gpu_device), gen)
    assert gen.get_state() == (3, 0)  # refused before anything is drawn
    handle.remove()
    mlp.run_layers(torch.randn(5, 64, device=gpu_device), gen)


def _decoder_and_edges(gpu_device):
    torch.manual_seed(6)
    mlp = MLP(in_features=64, latent_dimension=64, mlp_config=_decoder("layer", 0.3, "silu")).to(gpu_device).train()
    return mlp, torch.randn(300, 64, device=gpu_device), torch.arange(2000, device=gpu_device).view(2, 1000) % 300


def test_recomputed_modules_draw_their_ranges_again(gpu_device):
    """torch.utils.checkpoint around modules that take ranges themselves (decoder layers, edge dropout): with the generator's contexts the
    outputs, the gradients and the generator's state are those of the plain call, nested checkpoints too; without them the recomputation is
    refused instead of drawing another mask."""
    from amber_amd.mpn.common.edge_dropout import dropout_edge
    mlp, x, edges = _decoder_and_edges(gpu_device)
    gen = nd.CounterGenerator(12, device=gpu_device)
    check = torch.utils.checkpoint.checkpoint

    def layers(t):
        return mlp.run_layers(t, gen)

    def whole(t):
        _, kept = dropout_edge(edges, 0.4, True, gen)
        return layers(t) * kept[:300, None]

    def nested(t):
        return check(layers, check(whole, t, use_reentrant=False, context_fn=gen.checkpoint_contexts), use_reentrant=False,
                     context_fn=gen.checkpoint_contexts)

    def gradients(f):
        gen.set_state(12, 40)
        xl = x.clone().requires_grad_()
        y = f(xl)
        state = gen.get_state()
        return (y.detach(),) + torch.autograd.grad(y.square().sum(), [xl] + list(mlp.parameters())) + (state,)

    for f in (layers, whole, lambda t: layers(whole(t)), nested):
        plain = nested if f is nested else f
        want = gradients((lambda t: layers(whole(t))) if f is nested else f)
        got = gradients(nested if f is nested else lambda t: check(plain, t, use_reentrant=False, context_fn=gen.checkpoint_contexts))
        assert all(torch.equal(a, b) for a, b in zip(want[:-1], got[:-1])) and want[-1] == got[-1] == gen.get_state()
    both = lambda t: check(nested, t, use_reentrant=False, context_fn=gen.checkpoint_contexts)  # three deep
    assert all(torch.equal(a, b) for a, b in zip(want[:-1], gradients(both)[:-1]))
    for f in (layers, whole):
        for reentrant in (False, True):
            with pytest.raises(RuntimeError, match="checkpoint_contexts"):
                check(f, x.clone().requires_grad_(), use_reentrant=reentrant).sum().backward()
    gradients(layers)  # nothing is left open


def test_recomputed_model_draws_its_ranges_again(gpu_device):
    """The same around a whole SupervisedMPN: edge dropout and decoder dropout of one generator."""
    g = syn.grid_batch(num_graphs=2, nx=9, ny=8, in_node_features=5, in_edge_features=2).to(gpu_device)
    cfg = default_architecture(latent_dimension=64, num_steps=2)
    cfg["decoder"] = _decoder("layer", 0.2, "leakyrelu")
    torch.manual_seed(5)
    model = SupervisedMPN(AttrDict(cfg, dropout_generator="counter", dropout_seed=7), g).to(gpu_device).train()
    gen = model.mpn.dropout_generator
    anchor = torch.zeros((), device=gpu_device, requires_grad=True)  # something to differentiate among the checkpoint's arguments

    def step(**kw):
        gen.set_state(7, 9)
        f = lambda a: model(g) + a
        out = f(anchor) if not kw else torch.utils.checkpoint.checkpoint(f, anchor, use_reentrant=False, **kw)
        return (out.detach(),) + torch.autograd.grad(out.square().mean(), list(model.parameters()))

    want, got = step(), step(context_fn=gen.checkpoint_contexts)
    assert all(torch.equal(a, b) for a, b in zip(want, got)) and gen.get_state() == (7, 12)
    with pytest.raises(RuntimeError, match="checkpoint_contexts"):
        step(determinism_check="default")


def test_decoder_layers_with_leaky_relu_everywhere_but_at_the_kink(gpu_device):
    """MLP.run_layers with the default activation: the output in all rows, the gradient in every row none of whose pre-activations lies
    within 1e-5 of the kink (they are off by less: products of 64 terms of order 1, a few u sqrt(64)).  2e-5 of the largest value, as in
    test_decoder_layers_in_one_pass_each."""
    import copy
    torch.manual_seed(4)
    mlp = MLP(in_features=64, latent_dimension=64, mlp_config=_decoder("layer", 0.3, "leakyrelu")).to(gpu_device).train()
    with torch.no_grad():
        for q in mlp.parameters():
            q.add_(0.1 * torch.randn_like(q))
    x = torch.randn(700, 64, device=gpu_device, requires_grad=True)
    go = torch.randn(700, 64, device=gpu_device)
    ref = copy.deepcopy(mlp).cpu().double()
    y = mlp.run_layers(x, nd.CounterGenerator(31, device=gpu_device))
    dx, = torch.autograd.grad(y, x, go)
    t = xr = x.detach().cpu().double().requires_grad_()
    k, clear = 0, torch.ones(700, dtype=torch.bool)
    for layer in ref.mlp_layers:
        if isinstance(layer, torch.nn.Dropout):
            t = torch.where(orc.keep(t.numel(), 0.3, 31, k).view(t.shape), t / 0.7, torch.zeros((), dtype=torch.float64))
            k += 1
            continue
        if isinstance(layer, torch.nn.LeakyReLU):
            clear &= (t.detach().abs() > 1e-5).all(1)
        t = layer(t)
    want, = torch.autograd.grad(t, xr, go.cpu().double())
    assert int(clear.sum()) > 650
    assert float((y.detach().cpu().double() - t.detach()).abs().max()) <= 2e-5 * float(t.detach().abs().max())
    assert float((dx.cpu().double() - want)[clear].abs().max()) <= 2e-5 * float(want.abs().max())


@pytest.mark.parametrize("rows, width", [(4, 64), (63, 64), (20736, 64), (30011, 128), (6000, 1021), (3001, 8190), (2000, 16385)])
def test_weight_gradients_of_many_rows_lose_no_block(gpu_device, rows, width):
    """The sums over rows within the depth that they are added with: at least 256 blocks share the rows where there are many, a block's
    rows follow one another, then at most 64 additions join lanes, waves and blocks.  A block's sum missing or counted twice is far
    beyond that: every row adds g in [0.5, 1.5] to dbias, and as much times n to dweight."""
    x, w, b, go = _data(rows, width, torch.float32, torch.float32, seed=rows)
    go = go.clamp(-1, 1) / 2 + 1
    d = [t.to(gpu_device) for t in (x, w, b, go)]
    got = _run(d[0], None, d[1], d[2], True, 0.0, None, d[3])
    _compare(got, orc.tail(x, None, w, b, grad=go), _norm_bounds(x, w, b, go, chain=64 + rows // 256))
