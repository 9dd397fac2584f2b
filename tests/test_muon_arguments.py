"""Arguments and devices that the orthogonalising optimizer refuses before anything is launched or changed."""
import types

import pytest
import torch

from distributed_tensorflow_amd.ops import native as nv
from distributed_tensorflow_amd.optim import FlatMuon
from distributed_tensorflow_amd.runtime.arena import ParamArena, ParamSpec

SPECS = [ParamSpec("w", (12, 8), "trunc_normal"), ParamSpec("b", (8,), "zeros")]


def arena(device="cpu"):
    a = ParamArena(SPECS, device, FlatMuon.slots)
    a.initialize(1)
    return a


@pytest.mark.parametrize("eps", [0.0, -1e-7, float("nan")])
def test_flat_muon_refuses_an_eps_that_is_not_positive(eps):
    """With eps 0 a matrix whose gradient is zero would become 0 / 0."""
    with pytest.raises(ValueError, match="eps"):
        FlatMuon(arena(), ns_eps=eps)


@pytest.mark.gpu
def test_muon_step_refuses_an_eps_that_is_not_positive():
    a = arena("cuda")
    opt = FlatMuon(a)
    keep = a.params.clone()
    opt.step(0.1, vector_lr=0.0)   # no gradient: nothing moves
    assert torch.equal(a.params, keep)
    with pytest.raises(ValueError, match="eps"):
        nv.muon_step(a.params, a.grads, a.slots["m"], a.slots["v"], opt._hyper, opt._tables, nesterov=True, steps=5, eps=0.0)


def test_flat_muon_step_checks_the_device_before_it_launches(monkeypatch):
    """The scalars of a step go to the device by a launch of their own: on the wrong device nothing may be launched at all."""
    opt = FlatMuon(arena())
    launched = []

    def refuse(*tensors):
        raise ValueError("not on the current device")

    fake = types.SimpleNamespace(check_current_device=lambda what, *t: refuse(*t), set_scalars=lambda *a, **k: launched.append("set_scalars"),
                                 muon_step=lambda *a, **k: refuse())
    monkeypatch.setattr(opt, "_gpu", True)
    opt._nv, opt._hyper, opt._tables = fake, None, types.SimpleNamespace(workspace=None)
    with pytest.raises(ValueError, match="current device"):
        opt.step(0.1)
    assert launched == [] and opt.steps == 0


@pytest.mark.gpu
def test_flat_muon_step_on_another_device_launches_nothing(monkeypatch):
    """As if a second GPU were the current one."""
    a = arena("cuda")
    opt = FlatMuon(a)
    a.grads.fill_(1.0)
    keep = a.params.clone()
    launched = []
    monkeypatch.setattr(nv, "set_scalars", lambda *args, **kw: launched.append("set_scalars"))
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 1)
    with pytest.raises(ValueError, match="current device"):
        opt.step(0.1)
    assert launched == [] and opt.steps == 0 and torch.equal(a.params, keep)
