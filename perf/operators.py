"""Cases of the layer norm and dropout operators (amber_amd.norm_dropout) with their plain forms.

A case is one call as a training step or an inference makes it:

    norm   layer_norm over rows of features (forward alone, or forward and backward)
    drop   dropout from the counter-based generator
    tail   activate_norm_dropout: activation -> [LayerNorm] -> dropout, what follows every Linear of the decoder
    mask   keep_mask: which elements (the edges of a training step) the generator keeps

Random numbers are inputs: `state` holds (seed, offset) of the generator and element i's 32 bits are word i & 3 of
Philox-4x32-10 under key `seed` at counter (i >> 2, offset).
"""
import math

import torch

own = False

EPS = 1e-5
DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
M32 = 0xFFFFFFFF


def listed():
    return [
        # one refined mesh's vertices, inference: a single short call
        dict(name="norm_one_mesh", op="norm", rows=600, width=64, dtype="fp32", wdtype="fp32", train=False),
        # every node of the 10 M-edge batch (100 grids of 120 x 120 vertices), training
        dict(name="norm_batch_train", op="norm", rows=1440000, width=128, dtype="fp32", wdtype="fp32", train=True),
        # wide rows of odd length in 16 bits: no row starts where a vector does
        dict(name="norm_wide_odd_train", op="norm", rows=5003, width=4099, dtype="bf16", wdtype="bf16", train=True),
        # latents of one airfoil-sized batch
        dict(name="drop_airfoil_train", op="drop", rows=20736, width=64, dtype="fp32", p=0.1, train=True),
        # a large activation in 16 bits, forward alone
        dict(name="drop_wide", op="drop", rows=32768, width=4096, dtype="bf16", p=0.1, train=False),
        # one long row whose length is a prime
        dict(name="drop_prime_train", op="drop", rows=1, width=999983, dtype="fp16", p=0.5, train=True),
        # the decoder's layer on an airfoil-sized batch
        dict(name="tail_airfoil_train", op="tail", rows=20736, width=64, dtype="fp32", wdtype="fp32", act="leakyrelu", norm=True,
             p=0.1, train=True),
        # ... and on the 10 M-edge batch
        dict(name="tail_batch_train", op="tail", rows=1440000, width=128, dtype="fp32", wdtype="fp32", act="leakyrelu", norm=True,
             p=0.1, train=True),
        # a decoder without norm, smooth activation, odd width, 16 bits
        dict(name="tail_plain_odd_train", op="tail", rows=100003, width=333, dtype="fp16", wdtype="fp32", act="gelu", norm=False,
             p=0.2, train=True),
        # which edges of one airfoil-sized batch a training step keeps
        dict(name="mask_airfoil", op="mask", count=144002, p=0.1),
        # ... and of the 10 M-edge batch
        dict(name="mask_batch", op="mask", count=9984200, p=0.1),
    ]


def _log_int(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["norm", "norm", "drop", "drop", "tail", "tail", "mask"])
    p = round(rng.uniform(0.01, 0.7), 4)
    if op == "mask":
        return dict(op=op, count=_log_int(rng, 64, 9984200), p=p)
    width = rng.choice([32, 64, 128, 256]) if rng.random() < 0.3 else _log_int(rng, 1, 8192)
    rows = _log_int(rng, 1, min(1440000, 150000000 // width))
    dtype = rng.choice(list(DTYPES))
    case = dict(op=op, rows=rows, width=width, dtype=dtype, train=rng.random() < 0.7)
    if op != "drop":
        case["wdtype"] = rng.choice(["fp32", dtype])
    if op != "norm":
        case["p"] = p
    if op == "tail":
        case["act"] = rng.choice(["relu", "leakyrelu", "tanh", "elu", "silu", "mish", "gelu"])
        case["norm"] = rng.random() < 0.7
    return case


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _inputs(case, seed):
    gen = _generator(seed)
    dev = torch.device("cuda")
    s = {}
    if case["op"] != "norm":
        bits = torch.randint(0, 1 << 62, (2,), generator=gen, device=dev)
        s["state"] = torch.stack([bits[0], bits[1] >> 20])
    if case["op"] == "mask":
        return s
    rows, width, dtype = case["rows"], case["width"], DTYPES[case["dtype"]]
    x = torch.randn(rows, width, generator=gen, device=dev)
    if case["op"] != "drop":  # features with scales and offsets of their own
        x = x * (0.5 + torch.rand(width, generator=gen, device=dev)) + 0.5 * torch.randn(width, generator=gen, device=dev)
    s["x"] = x.to(dtype)
    if case["train"]:
        s["g"] = torch.randn(rows, width, generator=gen, device=dev).to(dtype)
    if case["op"] == "norm" or case.get("norm"):
        wdtype = DTYPES[case["wdtype"]]
        s["w"] = (1.0 + 0.2 * torch.randn(width, generator=gen, device=dev)).to(wdtype)
        s["b"] = (0.2 * torch.randn(width, generator=gen, device=dev)).to(wdtype)
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    if case.get("train"):
        for name in ("x", "w", "b"):
            if name in s:
                s[name].requires_grad_()
    s["case"] = case
    return s


def run(state):
    return _run_own(state) if own else _run_plain(state)


def _run_own(s):
    from amber_amd import norm_dropout as nd

    case = s["case"]
    if case["op"] == "mask":
        return nd.keep_mask(case["count"], case["p"], s["state"])
    with torch.set_grad_enabled(case["train"]):
        if case["op"] == "norm":
            y = nd.layer_norm(s["x"], s["w"], s["b"], eps=EPS)
        elif case["op"] == "drop":
            y = nd.dropout(s["x"], case["p"], s["state"])
        else:
            y = nd.activate_norm_dropout(s["x"], case["act"], s.get("w"), s.get("b"), normalize=case["norm"], eps=EPS, p=case["p"],
                                         state=s["state"])
    if not case["train"]:
        return y
    leaves = [s[k] for k in ("x", "w", "b") if k in s]
    return (y.detach(),) + torch.autograd.grad(y, leaves, s["g"])


# ---- plain form -----------------------------------------------------------------------------------------------------
def _random_words(n, state):
    """The generator's 32-bit words 0 .. n - 1 as int64."""
    seed, offset = state[0], state[1]
    group = torch.arange((n + 3) // 4, device=state.device)
    c0, c1 = group & M32, group >> 32
    c2 = (offset & M32).expand_as(group)
    c3 = ((offset >> 32) & M32).expand_as(group)
    k0, k1 = seed & M32, (seed >> 32) & M32
    for _ in range(10):
        p0, p1 = c0 * 0xD2511F53, c2 * 0xCD9E8D57  # modulo 2^64: both halves are right
        c0, c1, c2, c3 = ((p1 >> 32) & M32) ^ c1 ^ k0, p1 & M32, ((p0 >> 32) & M32) ^ c3 ^ k1, p0 & M32
        k0, k1 = (k0 + 0x9E3779B9) & M32, (k1 + 0xBB67AE85) & M32
    return torch.stack([c0, c1, c2, c3], dim=1).view(-1)[:n]


def _kept(n, p, state):
    return _random_words(n, state) >= int(p * 4294967296.0)


def _act(x, act):
    """(act(x), act'(x))"""
    one = torch.ones_like(x)
    if act == "relu":
        on = x > 0
        return torch.where(on, x, torch.zeros_like(x)), on.to(x.dtype)
    if act == "leakyrelu":
        slope = torch.where(x > 0, one, 0.01 * one)
        return x * slope, slope
    if act == "tanh":
        t = torch.tanh(x)
        return t, 1 - t * t
    if act == "elu":
        neg = torch.clamp(x, max=0)
        return torch.where(x > 0, x, torch.expm1(neg)), torch.where(x > 0, one, torch.exp(neg))
    sig = 1 / (1 + torch.exp(-x))
    if act == "silu":
        return x * sig, sig * (1 + x * (1 - sig))
    if act == "mish":
        t = torch.tanh(torch.where(x > 20, x, torch.log1p(torch.exp(torch.clamp(x, max=20)))))
        return x * t, t + x * sig * (1 - t * t)
    phi = 0.5 * (1 + torch.erf(x * math.sqrt(0.5)))
    return x * phi, phi + x * torch.exp(-0.5 * x * x) / math.sqrt(2 * math.pi)


@torch.no_grad()
def _run_plain(s):
    case = s["case"]
    if case["op"] == "mask":
        return _kept(case["count"], case["p"], s["state"])
    x = s["x"]
    v = x.float()
    normed = "w" in s
    if case["op"] == "tail":
        v, dact = _act(v, case["act"])
    if normed:
        w = s["w"].float()
        v = v - v.mean(1, keepdim=True)
        rstd = 1 / torch.sqrt((v * v).mean(1, keepdim=True) + EPS)
        n = v * rstd
        v = n * w + s["b"].float()
    if case["op"] != "norm":
        kept = _kept(v.numel(), case["p"], s["state"]).view(v.shape)
        scale = 1.0 / (1.0 - case["p"])
        v = torch.where(kept, v * scale, torch.zeros_like(v))
    y = v.to(x.dtype)
    if not case["train"]:
        return y
    g = s["g"].float()
    grads = ()
    if case["op"] != "norm":
        g = torch.where(kept, g * scale, torch.zeros_like(g))
    if normed:
        grads = ((g * n).sum(0).to(s["w"].dtype), g.sum(0).to(s["b"].dtype))
        h = g * w
        g = rstd * (h - h.mean(1, keepdim=True) - n * (h * n).mean(1, keepdim=True))
    if case["op"] == "tail":
        g = g * dact
    return (y, g.to(x.dtype)) + grads


# ---- in 64 bits -----------------------------------------------------------------------------------------------------
def _mul32(a, b):
    """(high, low) words of the product of a 32-bit tensor and a 32-bit constant, by 16-bit halves."""
    bl, bh = b & 0xFFFF, b >> 16
    al, ah = a % 65536, a // 65536
    low = al * bl
    mid = ah * bl + low // 65536
    mid2 = al * bh + mid % 65536
    return ah * bh + mid // 65536 + mid2 // 65536, (mid2 % 65536) * 65536 + low % 65536


def _exact_keep(n, p, state):
    seed, offset = (int(v) for v in state.tolist())
    limit = math.floor(p * 2.0 ** 32)
    keep = torch.empty((n + 3) // 4 * 4, dtype=torch.bool, device=state.device)
    step = 1 << 22
    for start in range(0, (n + 3) // 4, step):
        group = torch.arange(start, min(start + step, (n + 3) // 4), device=state.device)
        ctr = [group % 2 ** 32, group // 2 ** 32, torch.full_like(group, offset % 2 ** 32), torch.full_like(group, offset // 2 ** 32)]
        for rnd in range(10):
            k0 = (seed % 2 ** 32 + rnd * 0x9E3779B9) % 2 ** 32
            k1 = (seed // 2 ** 32 + rnd * 0xBB67AE85) % 2 ** 32
            hi0, lo0 = _mul32(ctr[0], 0xD2511F53)
            hi1, lo1 = _mul32(ctr[2], 0xCD9E8D57)
            ctr = [torch.bitwise_xor(torch.bitwise_xor(hi1, ctr[1]), k0), lo1, torch.bitwise_xor(torch.bitwise_xor(hi0, ctr[3]), k1), lo0]
        for word in range(4):
            keep[4 * start + word:4 * (start + len(group)):4] = ctr[word] >= limit
    return keep[:n]


def _exact_act(x, act):
    if act == "relu":
        return torch.relu(x)
    if act == "leakyrelu":
        return torch.nn.functional.leaky_relu(x, 0.01)
    if act == "tanh":
        return torch.tanh(x)
    if act == "elu":
        return torch.nn.functional.elu(x)
    if act == "silu":
        return x * torch.sigmoid(x)
    if act == "mish":
        return x * torch.tanh(torch.nn.functional.softplus(x, threshold=50))
    return x * 0.5 * torch.erfc(-x / math.sqrt(2.0))


def exact(case, seed):
    """The definition in float64; the gradients come from automatic differentiation of it."""
    s = _inputs(case, seed)
    if case["op"] == "mask":
        return None  # truth values: equal or not
    leaves = [s[k].double().requires_grad_(case["train"]) for k in ("x", "w", "b") if k in s]
    with torch.set_grad_enabled(case["train"]):
        y = leaves[0]
        if case["op"] == "tail":
            y = _exact_act(y, case["act"])
        if "w" in s:
            var, mean = torch.var_mean(y, dim=1, keepdim=True, correction=0)
            y = (y - mean) * torch.rsqrt(var + EPS) * leaves[1] + leaves[2]
        if case["op"] != "norm":
            y = y * _exact_keep(y.numel(), case["p"], s["state"]).view(y.shape) / (1.0 - case["p"])
    if not case["train"]:
        return y
    return (y.detach(),) + torch.autograd.grad(y, leaves, s["g"].double())


def work(case):
    if case["op"] == "mask":
        return {"bytes": 16 + case["count"], "flops": 0}
    n = case["rows"] * case["width"]
    size = torch.finfo(DTYPES[case["dtype"]]).bits // 8
    normed = case["op"] == "norm" or case.get("norm", False)
    nbytes = 2 * n * size
    flops = n * ((8 if normed else 0) + (1 if case["op"] != "norm" else 0) + (1 if case["op"] == "tail" else 0))
    if normed:
        nbytes += 2 * case["width"] * torch.finfo(DTYPES[case["wdtype"]]).bits // 8
    if case["train"]:
        nbytes *= 2  # the gradients of y, x and the weights
        flops += n * ((14 if normed else 0) + (1 if case["op"] != "norm" else 0) + (2 if case["op"] == "tail" else 0))
    return {"bytes": nbytes, "flops": flops}
