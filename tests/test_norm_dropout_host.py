"""CPU checks of the LayerNorm / dropout operators: the generator's published values, the oracle against torch's own layers, the
C entry points' and the Python wrappers' refusals, the wiring of the `dropout_generator` config.  Nothing runs on a GPU."""
import ctypes as C
import math

import numpy as np
import pytest
import torch
import torch.multiprocessing as mp

from amber_amd import _lib, norm_dropout as nd, synthetic as syn
from amber_amd.architecture.mlp import MLP
from amber_amd.architecture.supervised_mpn import SupervisedMPN
from amber_amd.config import AttrDict, default_architecture
from oracle import norm_dropout_oracle as orc


@pytest.mark.parametrize("counter, key, want", [
    # known answers published with the generator: zeros, all bits set, digits of pi
    ((0, 0, 0, 0), (0, 0), (0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8)),
    ((0xFFFFFFFF,) * 4, (0xFFFFFFFF,) * 2, (0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD)),
    ((0x243F6A88, 0x85A308D3, 0x13198A2E, 0x03707344), (0xA4093822, 0x299F31D0), (0xD16CFE09, 0x94FDCCEB, 0x5001E420, 0x24126EA1)),
])
def test_oracle_generator_known_answers(counter, key, want):
    assert tuple(int(v) for v in orc.philox(np.array(counter, dtype=np.uint32), key)) == want


def test_oracle_words_are_one_sequence():
    full = orc.words(0, 1000, 7, 3)
    for start, count in ((0, 1), (1, 5), (3, 997), (510, 7), (999, 1)):
        assert np.array_equal(orc.words(start, count, 7, 3), full[start:start + count])
    assert not np.array_equal(orc.words(0, 100, 7, 4), full[:100])
    # mean of n fair draws: standard deviation sqrt(p (1 - p) / n) = 0.0009; five of them
    assert abs(float(orc.keep(100000, 0.1, 11, 5).double().mean()) - 0.9) < 5 * math.sqrt(0.09 / 100000)


@pytest.mark.parametrize("act", [None, "relu", "leakyrelu", "tanh", "elu", "silu", "mish", "gelu"])
def test_oracle_tail_equals_torch_layers(act):
    g = torch.Generator().manual_seed(1)
    x, go = (torch.randn(5, 12, generator=g, dtype=torch.float64) for _ in range(2))
    w, b = (torch.randn(12, generator=g, dtype=torch.float64) for _ in range(2))
    xr, wr, br = (t.clone().requires_grad_() for t in (x, w, b))
    want = torch.nn.functional.layer_norm(orc.act(xr, act), (12,), wr, br, 1e-5)
    grads = torch.autograd.grad(want, (xr, wr, br), go)
    for got, ref in zip(orc.tail(x, act, w, b, grad=go), (want.detach(),) + grads):
        assert torch.allclose(got, ref, rtol=1e-12, atol=1e-12)


def _tail_desc(**kw):
    base = dict(dtype=0, weight_dtype=0, activation=-1, normalize=1, p=0.0, eps=1e-5, sequence=0)
    base.update(kw)
    return _lib.AmberTailDesc(**base)


@pytest.mark.parametrize("kw, rows, width, code, message", [
    (dict(dtype=3), 4, 8, -2, b"dtype id 3"),
    (dict(dtype=1, weight_dtype=2), 4, 8, -2, b"weight_dtype id 2"),
    (dict(activation=7), 4, 8, -2, b"activation id 7"),
    (dict(activation=-2), 4, 8, -2, b"activation id -2"),
    (dict(p=-0.1), 4, 8, -1, b"between 0 and 1"),
    (dict(p=1.5), 4, 8, -1, b"between 0 and 1"),
    (dict(p=float("nan")), 4, 8, -1, b"between 0 and 1"),
    (dict(eps=-1.0), 4, 8, -1, b"eps"),
    (dict(eps=float("nan")), 4, 8, -1, b"eps"),
    (dict(eps=float("inf")), 4, 8, -1, b"eps"),
    (dict(sequence=-1), 4, 8, -1, b"sequence"),
    ({}, -1, 8, -1, b"negative size"),
    ({}, 4, -8, -1, b"negative size"),
    ({}, 4, 0, -1, b"no features"),
    ({}, 1 << 40, 1 << 20, -1, b"out of range"),
    ({}, 1, (1 << 30) + 1, -1, b"out of range"),
    (dict(normalize=0), 1, (1 << 50) + 1, -1, b"out of range"),
    (dict(p=0.5), 4, 8, -1, b"state is NULL"),
    ({}, 4, 8, -1, b"x / y is NULL"),
])
def test_c_forward_refusals(kw, rows, width, code, message):
    lib = _lib.load()
    rc = lib.amber_mpn_tail_forward(C.byref(_tail_desc(**kw)), rows, width, 0, width, 0, 0, 0, 0, 0, 0)
    assert rc == code and message in lib.amber_mpn_last_error()


def test_c_refusals_that_need_pointers_never_launch():
    """Host pointers stand in for device ones: every call below is refused before anything is launched."""
    lib = _lib.load()
    buf = (C.c_char * 4096)()
    p = C.addressof(buf)
    d = C.byref(_tail_desc())
    plain = C.byref(_tail_desc(normalize=0, activation=1))
    assert lib.amber_mpn_tail_forward(None, 4, 8, p, 8, 0, 0, 0, p, 0, 0) == -1
    assert lib.amber_mpn_tail_forward(d, 4, 8, p, -8, 0, 0, 0, p, 0, 0) == -1
    assert lib.amber_mpn_tail_forward(d, 4, 8, p, 1 << 50, 0, 0, 0, p, 0, 0) == -1
    assert lib.amber_mpn_tail_forward(plain, 4, 8, p, 9, 0, 0, 0, p, 0, 0) == -2  # strided rows
    assert lib.amber_mpn_tail_forward(plain, 4, 8, p, 8, p, 0, 0, p, 0, 0) == -1  # weight without normalize
    assert lib.amber_mpn_tail_forward(plain, 4, 8, p, 8, 0, p, 0, p, 0, 0) == -1
    back = lib.amber_mpn_tail_backward
    need = lib.amber_mpn_tail_backward_workspace_bytes(d, 4000, 8)
    assert need >= 2 * 8 * 4 and lib.amber_mpn_tail_backward_workspace_bytes(d, 4, 8) == 0
    assert back(d, 4, 8, p, 8, 0, 8, 0, p, 0, p, 0, 0, 0, 0, 0) == -1  # grad_y
    assert back(d, 4, 8, 0, 8, p, 8, 0, p, 0, p, 0, 0, 0, 0, 0) == -1  # x
    assert back(d, 4, 8, p, 8, p, 8, 0, 0, 0, p, 0, 0, 0, 0, 0) == -1  # stats
    assert back(d, 4, 8, p, 8, p, -1, 0, p, 0, p, 0, 0, 0, 0, 0) == -1
    assert back(d, 4000, 8, p, 8, p, 8, 0, p, 0, p, p, 0, 0, 0, 0) == -1  # workspace
    assert back(d, 4000, 8, p, 8, p, 8, 0, p, 0, p, p, 0, p, need - 1, 0) == -3
    assert back(plain, 4, 8, 0, 8, p, 8, 0, 0, 0, p, 0, 0, 0, 0, 0) == -1  # the activation needs x
    assert back(plain, 4, 8, p, 8, p, 9, 0, 0, 0, p, 0, 0, 0, 0, 0) == -2
    assert back(plain, 4, 8, p, 8, p, 8, 0, 0, 0, p, p, 0, 0, 0, 0) == -1  # grad_weight without normalize
    assert lib.amber_mpn_tail_backward_workspace_bytes(C.byref(_tail_desc(p=2.0)), 4, 8) == 0
    assert lib.amber_mpn_generator_take(0, 1, p, 0) == -1 and lib.amber_mpn_generator_take(p, -1, p, 0) == -1
    assert lib.amber_mpn_keep_mask(p, 0, 2.0, 4, p, 0) == -1 and lib.amber_mpn_keep_mask(p, -1, 0.5, 4, p, 0) == -1
    assert lib.amber_mpn_keep_mask(0, 0, 0.5, 4, p, 0) == -1 and lib.amber_mpn_keep_mask(p, 0, 0.5, 4, 0, 0) == -1
    assert lib.amber_mpn_keep_mask(p, 0, 0.5, -4, p, 0) == -1


def test_c_calls_with_nothing_to_do():
    lib = _lib.load()
    d = C.byref(_tail_desc(p=0.5))
    assert lib.amber_mpn_tail_forward(d, 0, 8, 0, 8, 0, 0, 0, 0, 0, 0) == 0
    assert lib.amber_mpn_tail_forward(C.byref(_tail_desc(normalize=0, p=0.5)), 5, 0, 0, 0, 0, 0, 0, 0, 0, 0) == 0
    assert lib.amber_mpn_tail_backward(d, 0, 8, 0, 8, 0, 8, 0, 0, 0, 0, 0, 0, 0, 0, 0) == 0
    assert lib.amber_mpn_keep_mask(0, 0, 0.5, 0, 0, 0) == 0


def test_python_refuses_cpu_tensors():
    x = torch.zeros(3, 4)
    state = torch.zeros(2, dtype=torch.int64)
    for call in (lambda: nd.layer_norm(x), lambda: nd.dropout(x, 0.1, state), lambda: nd.activate_norm_dropout(x, "relu"),
                 lambda: nd.keep_mask(3, 0.1, state), lambda: nd.CounterGenerator(1).take()):
        with pytest.raises(RuntimeError, match="MI355X only"):
            call()


def test_python_checks():
    """Everything but the device is checked first, so a CPU tensor shows the refusals."""
    x = torch.zeros(3, 4, dtype=torch.bfloat16)
    state = torch.zeros(2, dtype=torch.int64)
    for p in (-0.1, 1.1, float("nan")):
        for call in (lambda: nd.dropout(x, p, state), lambda: nd.keep_mask(4, p, state), lambda: nd.activate_norm_dropout(x, None, p=p)):
            with pytest.raises(ValueError, match="between 0 and 1"):
                call()
    for call in (lambda: nd.dropout(x, 0.5), lambda: nd.keep_mask(4, 0.5, None), lambda: nd.activate_norm_dropout(x, None, p=0.5)):
        with pytest.raises(ValueError, match="needs the generator"):
            call()
    for bad in (torch.zeros(2), torch.zeros(3, dtype=torch.int64), torch.zeros(2, 2, dtype=torch.int64)[:, 0],
                torch.zeros(1, 2, dtype=torch.int64)):
        for call in (lambda: nd.dropout(x, 0.5, bad), lambda: nd.keep_mask(4, 0.5, bad)):
            with pytest.raises(ValueError, match="contiguous int64"):
                call()
    for bad in (-1, 1 << 62):
        for call in (lambda: nd.dropout(x, 0.5, state, sequence=bad), lambda: nd.keep_mask(4, 0.5, state, bad)):
            with pytest.raises(ValueError, match="sequence"):
                call()
    for bad in (-1e-5, float("nan"), float("inf")):
        with pytest.raises(ValueError, match="eps"):
            nd.layer_norm(x, eps=bad)
    with pytest.raises(ValueError, match="weight of shape"):
        nd.layer_norm(x, torch.ones(3))
    with pytest.raises(ValueError, match="bias of shape"):
        nd.layer_norm(x, None, torch.ones(1, 4))
    with pytest.raises(TypeError, match="x's type"):
        nd.layer_norm(x, torch.ones(4, dtype=torch.float16))
    with pytest.raises(TypeError, match="weight is"):
        nd.layer_norm(x, torch.ones(4), torch.ones(4, dtype=torch.bfloat16))
    with pytest.raises(ValueError, match="is on"):
        nd.layer_norm(x, torch.ones(4, device="meta"))
    for bad in (torch.tensor(1.0), torch.zeros(3, 0)):
        with pytest.raises(ValueError, match="last dimension"):
            nd.layer_norm(bad)
    for bad in (x.double(), x.long(), x.bool()):
        with pytest.raises(TypeError, match="float32, bfloat16 or float16"):
            nd.layer_norm(bad)
    with pytest.raises(ValueError, match="Unknown activation"):
        nd.activate_norm_dropout(x, "swiglu")
    with pytest.raises(ValueError, match="without normalize"):
        nd.activate_norm_dropout(x, "relu", torch.ones(4), normalize=False)
    with pytest.raises(ValueError, match="elements"):
        nd.keep_mask(-1, 0.5, state)
    for bad in (0, -1, 1 << 62):
        with pytest.raises(ValueError, match="ranges"):
            nd.CounterGenerator(1).take(bad)


def test_generator_state_round_trip():
    gen = nd.CounterGenerator((1 << 64) - 3)
    assert gen.get_state() == ((1 << 64) - 3, 0) and not gen.state_dict()
    gen.set_state(5, (1 << 63) + 9)
    assert gen.get_state() == (5, (1 << 63) + 9)
    torch.manual_seed(77)
    assert nd.CounterGenerator().get_state() == (77, 0)


def test_dropout_generator_config():
    g = syn.grid_batch(num_graphs=1, nx=5, ny=4)
    cfg = default_architecture(latent_dimension=32, num_steps=1)
    keys = set(SupervisedMPN(cfg, g).state_dict())
    assert SupervisedMPN(cfg, g).mpn.dropout_generator is None
    model = SupervisedMPN(AttrDict(cfg, dropout_generator="counter", dropout_seed=9), g)
    assert set(model.state_dict()) == keys  # checkpoints load either way
    assert model.mpn.maybe_edge_dropout.generator is model.mpn.dropout_generator
    assert model.mpn.dropout_generator.get_state() == (9, 0)
    assert SupervisedMPN(AttrDict(cfg, dropout_generator="torch"), g).mpn.dropout_generator is None
    with pytest.raises(ValueError, match="dropout_generator"):
        SupervisedMPN(AttrDict(cfg, dropout_generator="philox"), g)


def test_decoder_layers_without_a_generator_are_the_modules():
    cfg = AttrDict({"activation_function": "tanh", "num_layers": 2,
                    "regularization": {"dropout": 0.0, "spectral_norm": False, "latent_normalization": "layer"}})
    mlp = MLP(in_features=8, latent_dimension=8, mlp_config=cfg)
    x = torch.randn(4, 8)
    want = x
    for layer in mlp.mlp_layers:
        want = layer(want)
    assert torch.equal(mlp.run_layers(x), want)


def _broadcast_worker(rank, port, ret):
    import os

    import torch.distributed as dist

    from amber_amd import sharding
    os.environ.update(MASTER_ADDR="127.0.0.1", MASTER_PORT=str(port))
    dist.init_process_group("gloo", rank=rank, world_size=2)
    module = torch.nn.Sequential(torch.nn.BatchNorm1d(3), nd.CounterGenerator(40 + rank))
    module[0].running_mean.fill_(float(rank + 1))
    sharding.broadcast_buffers(module, src=0)
    ret[rank] = (module[0].running_mean.tolist(), module[1].get_state())
    dist.barrier()
    dist.destroy_process_group()


def test_world_size_2_broadcast_leaves_each_rank_its_generator():
    import socket
    with socket.socket() as s:
        s.bind(("127.0.0.1", 0))
        port = s.getsockname()[1]
    ret = mp.Manager().dict()
    mp.spawn(_broadcast_worker, args=(port, ret), nprocs=2, join=True)
    assert ret[0] == ([1.0] * 3, (40, 0)) and ret[1] == ([1.0] * 3, (41, 0))


def test_taking_anew_inside_a_backward_pass_is_refused():
    gen = nd.CounterGenerator(3)

    class Again(torch.autograd.Function):
        @staticmethod
        def forward(ctx, x):
            return x * 2

        @staticmethod
        def backward(ctx, g):
            gen.take_in_module()

    with pytest.raises(RuntimeError, match="checkpoint_contexts"):
        Again.apply(torch.ones(2, requires_grad=True)).sum().backward()
    first, again = gen.checkpoint_contexts()
    with again, pytest.raises(RuntimeError, match="other ranges"):  # more than the first pass took
        gen.take()
    with first, pytest.raises(RuntimeError, match="MI355X only"):  # the generator itself is asked
        gen.take()


def test_drawing_dropout_with_hooks_is_refused():
    cfg = AttrDict({"activation_function": "tanh", "num_layers": 1,
                    "regularization": {"dropout": 0.5, "spectral_norm": False, "latent_normalization": None}})
    mlp = MLP(in_features=8, latent_dimension=8, mlp_config=cfg)
    mlp.mlp_layers[2].register_forward_pre_hook(lambda mod, args: None)
    with pytest.raises(RuntimeError, match="dropout_generator"):
        mlp.run_layers(torch.randn(4, 8), nd.CounterGenerator(1))
