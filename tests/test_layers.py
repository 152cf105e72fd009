"""CPU tests of the layer operators: the C ABI of include/az_layers.h, the refusals of every entry point (none
of which reaches a GPU)."""
import ctypes as C
import os
import re

import pytest
import torch

import alphazero_amd as mctx
from alphazero_amd import _native as nat

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_library_exports_every_declared_layer_symbol():
    header = open(os.path.join(ROOT, "include", "az_layers.h")).read()
    header = re.sub(r"/\*.*?\*/", "", header, flags=re.S)
    declared = set(re.findall(r"\b(az_[a-z_0-9]+)\s*\(", header))
    assert declared == set(nat.LAYER_SIGNATURES), declared ^ set(nat.LAYER_SIGNATURES)
    for name in declared:
        assert hasattr(nat.lib(), name)
    assert C.sizeof(nat.SampleDesc) == 4 * 4 + 3 * 8 + 7 * 8


F, H = torch.float32, torch.float16


def t(*shape, dtype=F):
    return torch.zeros(shape, dtype=dtype)


@pytest.mark.parametrize("error,args,kw", [
    (ValueError, (t(3, 4), t(5, 2)), {}),                                   # fan_in
    (ValueError, (t(3, 4), t(4)), {}),
    (ValueError, (t(3, 0), t(0, 2)), {}),
    (ValueError, (t(3, 4), t(4, 0)), {}),
    (ValueError, (t(3, 4), t(4, 2)), dict(bias=t(3))),
    (ValueError, (t(3, 4), t(4, 2)), dict(bias=t(1, 2))),
    (ValueError, (t(3, 4), t(4, 2)), dict(residual=t(1, 2))),               # no broadcasting
    (ValueError, (t(3, 4), t(4, 2)), dict(residual=t(3, 4))),
    (ValueError, (t(3, 4), t(4, 2)), dict(activation="tanh")),
    (TypeError, (t(3, 4), t(4, 2, dtype=H)), {}),
    (TypeError, (t(3, 4), t(4, 2)), dict(bias=t(2, dtype=H))),
    (TypeError, (t(3, 4), t(4, 2)), dict(residual=t(3, 2, dtype=H))),
    (TypeError, (t(3, 4, dtype=torch.float64), t(4, 2, dtype=torch.float64)), {}),
    (ValueError, (t(3, 4), t(4, 2).to("meta")), {}),                        # another device
    (NotImplementedError, (t(3, 4), t(4, 2)), {}),                          # no CPU path
])
def test_dense_refusals(error, args, kw):
    with pytest.raises(error):
        mctx.dense(*args, **kw)


@pytest.mark.parametrize("error,args,kw", [
    (ValueError, (t(3, 0),), {}),
    (ValueError, (torch.tensor(1.0),), {}),
    (ValueError, (t(3, 4), t(3)), {}),
    (ValueError, (t(3, 4),), dict(bias=t(1, 4))),
    (ValueError, (t(3, 4),), dict(eps=-1.0)),
    (ValueError, (t(3, 4),), dict(eps=float("nan"))),
    (TypeError, (t(3, 4), t(4, dtype=H)), {}),
    (TypeError, (t(3, 4, dtype=H), t(4, dtype=H), t(4)), {}),               # scale and bias of two types
    (TypeError, (t(3, 4, dtype=torch.int32),), {}),
    (NotImplementedError, (t(3, 4),), {}),
])
def test_layer_norm_refusals(error, args, kw):
    with pytest.raises(error):
        mctx.layer_norm(*args, **kw)


@pytest.mark.parametrize("error,args,kw", [
    (ValueError, (t(4), t(4)), {}),
    (ValueError, (t(4, 0), t(4)), {}),
    (ValueError, (t(4, 3), t(3)), {}),
    (ValueError, (t(4, 3), t(4, dtype=H)), {}),
    (TypeError, (t(4, 3, dtype=torch.float64), t(4)), {}),
    (ValueError, (t(4, 3), t(4)), dict(invalid_actions=t(3))),
    (ValueError, (t(4, 3), t(4)), dict(temperature=-1.0)),
    (ValueError, (t(4, 3), t(4)), dict(temperature=float("nan"))),
    (ValueError, (t(4, 3), t(4)), dict(temperature=float("inf"))),
    (ValueError, (t(4, 3), t(4)), dict(temperature=t(3))),
    (ValueError, (t(4, 3), t(4)), dict(top_k=-1)),
    (ValueError, (t(4, 3), t(4)), dict(top_k=1.5)),
    (ValueError, (t(4, 3), t(4)), dict(top_p=1.5)),
    (ValueError, (t(4, 3), t(4)), dict(min_p=-0.1)),
    (ValueError, (t(4, 3), t(4)), dict(min_p=t(4, 1))),
    (ValueError, (t(4, 3), t(4)), dict(top_p=t(4).to("meta"))),
    (NotImplementedError, (t(4, 3), t(4)), {}),
])
def test_sample_actions_refusals(error, args, kw):
    with pytest.raises(error):
        mctx.sample_actions(*args, **kw)


def test_native_refusals():
    """The C entry points refuse before they launch (all pointers here are null or never read)."""
    lib = nat.lib()
    some = C.c_void_p(4096)
    assert lib.az_dense_workspace_bytes(3, 4, 4, 4, 0) == -1
    assert lib.az_dense_workspace_bytes(0, -1, 4, 4, 0) == -1
    assert lib.az_dense_workspace_bytes(0, 4, 0, 4, 0) == -1
    assert lib.az_dense_workspace_bytes(0, 4, 4, 2 ** 20 + 1, 0) == -1
    assert lib.az_dense_workspace_bytes(0, 2 ** 31 - 1, 4, 4, 0) == -1
    assert lib.az_dense_workspace_bytes(0, 4, 4, 4, 2) == -1
    assert lib.az_dense_workspace_bytes(0, 0, 4, 4, 1) == 0
    dense = lib.az_dense_forward
    assert dense(0, 9, 4, 4, 4, some, some, None, None, some, None, some, 1 << 30, None) == -1
    assert dense(0, 0, 4, 4, 4, None, some, None, None, some, None, some, 1 << 30, None) == -1
    assert dense(0, 0, 0, 4, 4, None, None, None, None, None, None, None, 0, None) == 0      # no rows
    n = lib.az_dense_workspace_bytes(0, 256, 4096, 4096, 0)
    assert n > 0
    assert dense(0, 0, 256, 4096, 4096, some, some, None, None, some, None, some, n - 1, None) == -1
    assert dense(0, 0, 256, 4096, 4096, some, some, None, None, some, None, None, n, None) == -1
    assert dense(0, 0, 256, 4096, 4096, some, some, None, None, some, None, C.c_void_p(4100), n, None) == -1
    back = lib.az_dense_backward
    assert back(0, 1, 4, 4, 4, some, some, None, some, some, some, some, some, 1 << 30, None) == -1   # z is missing
    assert back(0, 0, 4, 4, 4, None, some, None, some, some, some, some, some, 1 << 30, None) == -1
    assert back(0, 0, 4, 4, 4, some, some, None, some, None, None, None, None, 0, None) == 0          # nothing asked
    assert lib.az_layer_norm_workspace_bytes(4, 0) == -1
    norm = lib.az_layer_norm_forward
    assert norm(0, 1, 4, 4, some, some, some, 1e-6, some, None, None, None) == -1            # parameter type
    assert norm(0, 0, 4, 4, some, some, some, 1e-6, some, some, None, None) == -1            # mean without rstd
    assert norm(0, 0, 4, 2 ** 20 + 1, some, some, some, 1e-6, some, None, None, None) == -2
    assert lib.az_layer_norm_backward(0, 0, 4, 4, some, some, some, some, some, some, some, some, None, 0, None) == -1
    d = nat.SampleDesc(dtype=0, rows=4, actions=0)
    assert lib.az_sample_actions(C.byref(d), some, some, None) == -1
    d.actions = 2 ** 20 + 1
    assert lib.az_sample_actions(C.byref(d), some, some, None) == -2
    d.actions = 4
    assert lib.az_sample_actions(C.byref(d), some, some, None) == -1
    d.rows = 0
    assert lib.az_sample_actions(C.byref(d), None, None, None) == 0


def test_sample_actions_refuses_fractional_counts():
    with pytest.raises(TypeError, match="top_k"):
        mctx.sample_actions(t(4, 3), t(4), top_k=torch.full((4,), 1.5))


def test_prior_policy_and_networks_refusals():
    from alphazero_amd import networks, trainer
    root = mctx.RootFnOutput(prior_logits=t(4, 3), value=t(4), embedding=None)
    with pytest.raises(NotImplementedError):       # no CPU path
        mctx.prior_policy((), 0, root, uniform=t(4))
    with pytest.raises(ValueError):
        mctx.prior_policy((), 0, root, uniform=t(3))
    nets = networks.ResidualNetworks(12, 3, width=8, blocks=2, device="cpu")
    assert len(nets.leaves()) == 2 + 2 * 6 + 2 + 2 + 2
    with pytest.raises(ValueError):
        nets.forward(t(4, 5))
    with pytest.raises(ValueError):
        nets.forward(t(3, 3, 5))                   # 15 values, not 12
    with pytest.raises(NotImplementedError):
        nets.forward(t(4, 3, 4))
    with pytest.raises(ValueError):
        trainer.Trainer(trainer.Config(env_id="Breakout-MinAtar", torso="transformer"), device="cpu")
    # what the learner computes without the operators is what it computed before
    assert trainer.Config().native_dense is False and trainer.Config().torso == "conv"


def test_sizes_beyond_the_abi_are_refused():
    """Rows and widths are 32-bit numbers there: tensors (without storage here) that would wrap."""
    big = torch.empty((1,), dtype=H).expand(2 ** 32 + 5, 1)
    with pytest.raises(NotImplementedError):
        mctx.dense(big, t(1, 1, dtype=H))
    with pytest.raises(NotImplementedError):
        mctx.layer_norm(big)
    with pytest.raises(NotImplementedError):
        mctx.sample_actions(big, torch.empty((1,)).expand(2 ** 32 + 5))
    from alphazero_amd import layers
    with pytest.raises(NotImplementedError, match="rows or columns"):
        layers._rows(big)
    lib = nat.lib()
    some = C.c_void_p(4096)
    # more outputs or rows than a launch has threads for
    assert lib.az_dense_forward(1, 0, 2 ** 31 - 2 ** 16, 1, 2 ** 20, some, some, None, None, some, None, some, 1 << 62, None) == -2
    d = nat.SampleDesc(dtype=0, rows=2 ** 31 - 1, actions=2, logits=4096, uniform=4096)
    assert lib.az_sample_actions(C.byref(d), some, some, None) == -2


def test_dual_tensors_are_refused():
    """Forward-mode differentiation: the tangent is not dropped silently, whichever tensor carries it."""
    import torch.autograd.forward_ad as forward_ad
    x, w, b = torch.ones(3, 4), torch.ones(4, 2), torch.ones(2)
    with forward_ad.dual_level():
        def dual(v):
            return forward_ad.make_dual(v, torch.ones_like(v))
        for args, kw in (((dual(x), w), {}), ((x, dual(w)), {}), ((x, w, dual(b)), {}), ((x, w), dict(residual=dual(t(3, 2)))),
                         ((dual(x).reshape(1, 3, 4), w), {})):
            with pytest.raises(NotImplementedError, match="forward-mode"):
                mctx.dense(*args, **kw)
        for args in ((dual(x),), (x, dual(t(4))), (x, t(4), dual(t(4)))):
            with pytest.raises(NotImplementedError, match="forward-mode"):
                mctx.layer_norm(*args)
        with torch.no_grad(), pytest.raises(NotImplementedError, match="forward-mode"):
            mctx.dense(dual(x), w)
        with pytest.raises(NotImplementedError, match="on the GPU"):      # none of them is dual
            mctx.dense(x, w, b)
    with pytest.raises(NotImplementedError, match="forward-mode"):
        torch.func.jvp(lambda v: mctx.dense(v, w), (x,), (x,))


@pytest.mark.parametrize("call", [lambda v: mctx.dense(v, t(4, 2)), lambda v: mctx.layer_norm(v),
                                  lambda v: mctx.sample_actions(v, t(3))[0]], ids=["dense", "layer_norm", "sample_actions"])
def test_recorded_calls_are_refused(call):
    """A trace would hold the outputs' allocation and nothing that writes them."""
    from torch.fx.experimental.proxy_tensor import make_fx
    x = torch.ones(3, 4)
    with pytest.raises(NotImplementedError, match="traced"):
        torch.jit.trace(call, (x,))
    for mode in ("real", "fake"):
        with pytest.raises(NotImplementedError, match="traced"):
            make_fx(call, tracing_mode=mode)(x)
    with pytest.raises(NotImplementedError, match="on the GPU"):
        call(x)


def test_dual_output_gradients_are_refused(monkeypatch):
    """The same for the backward passes (without their native calls, which this machine need not be able to make)."""
    import torch.autograd.forward_ad as forward_ad
    from alphazero_amd import layers
    monkeypatch.setattr(layers, "_checked", lambda *args: None)
    monkeypatch.setattr(layers, "_native", lambda *args: None)
    x, w = torch.ones(3, 4, requires_grad=True), torch.ones(4, 4)
    for y in (mctx.dense(x, w), mctx.layer_norm(x)):
        torch.autograd.grad(y, x, torch.ones(3, 4), retain_graph=True)
        with forward_ad.dual_level(), pytest.raises(NotImplementedError, match="forward-mode"):
            torch.autograd.grad(y, x, forward_ad.make_dual(torch.ones(3, 4), torch.ones(3, 4)))


@pytest.mark.parametrize("match,kw", [
    ("native_dense", dict(env_id="Breakout-MinAtar", native_dense=True)),
    ("has no torso", dict(env_id="CartPole-v1", torso="residual")),
    ("neither", dict(env_id="CartPole-v1", torso="transformer")),
])
def test_trainer_refuses_settings_without_effect(match, kw):
    from alphazero_amd import trainer
    with pytest.raises(ValueError, match=match):
        trainer.Trainer(trainer.Config(**kw), device="cpu")
