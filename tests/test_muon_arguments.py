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
