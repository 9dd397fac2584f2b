"""A FlatMuon step captured into a graph, and its launches recorded into a step program, against the same steps taken eagerly."""
import pytest
import torch

from distributed_tensorflow_amd.ops import native as nv
from distributed_tensorflow_amd.optim import FlatMuon
from distributed_tensorflow_amd.runtime.arena import ParamArena, ParamSpec

# matrices only: the scalars of a step are part of it, and the vectors' Adam step size changes from step to step
SPECS = [ParamSpec("small", (40, 24), "trunc_normal"), ParamSpec("tall", (300, 70), "trunc_normal"), ParamSpec("wide", (70, 900), "trunc_normal")]


def arena():
    a = ParamArena(SPECS, "cuda", FlatMuon.slots)
    a.initialize(3)
    return a


def gradient(total, seed):
    return 1e-3 * torch.randn(total, device="cuda", generator=torch.Generator(device="cuda").manual_seed(seed))


@pytest.mark.gpu
@pytest.mark.parametrize("products", nv.PRODUCTS)
def test_a_captured_step_replays(products):
    held, twin = arena(), arena()
    captured, eager = FlatMuon(held, weight_decay=0.1, ns_products=products), FlatMuon(twin, weight_decay=0.1, ns_products=products)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    keep = held.params.clone()
    with torch.cuda.stream(side):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            captured.step(0.02, grad_scale=0.5)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(held.params, keep)
    for seed in range(3):
        g = gradient(held.total, seed)
        held.grads.copy_(g)
        twin.grads.copy_(g)
        graph.replay()
        eager.step(0.02, grad_scale=0.5)   # in between, on workspace of its own
        torch.cuda.synchronize()
        assert torch.equal(held.params, twin.params) and torch.equal(held.slots["m"], twin.slots["m"])


@pytest.mark.gpu
@pytest.mark.parametrize("products", nv.PRODUCTS)
def test_recorded_launches_run(products):
    """The scalars of a step are no part of a program, which refuses them: they are set before each run, as for the other optimizers."""
    held, twin = arena(), arena()
    recorded, eager = FlatMuon(held, ns_products=products), FlatMuon(twin, ns_products=products)
    out = torch.zeros(300, 70, device="cuda")
    ws = torch.empty(nv.newton_schulz_workspace(300, 70, products=products), device="cuda", dtype=torch.uint8)
    keep, prog = held.params.clone(), nv.hip().Program()
    prog.begin_record()
    try:
        with pytest.raises(RuntimeError, match="cannot be recorded"):
            recorded.step(0.02)
        nv.muon_step(held.params, held.grads, held.slots["m"], held.slots["v"], recorded._hyper, recorded._tables, nesterov=True, steps=5)
        with pytest.raises(ValueError, match="workspace"):
            nv.newton_schulz(held.grad("tall"), out=out, products=products)
        nv.newton_schulz(held.grad("tall"), out=out, products=products, workspace=ws)
    finally:
        prog.end_record()
    torch.cuda.synchronize()
    assert torch.equal(held.params, keep) and not out.any()
    for seed in range(2):
        g = gradient(held.total, 10 + seed)
        held.grads.copy_(g)
        twin.grads.copy_(g)
        nv.set_scalars(recorded._hyper, (0.02, 0.95, 1.0, 1.0, 0.0, 0.1, 0.001, 1e-8))
        prog.run(torch.cuda.current_stream().cuda_stream, -1)
        eager.step(0.02)
        torch.cuda.synchronize()
        assert torch.equal(held.params, twin.params) and torch.equal(out, nv.newton_schulz(twin.grad("tall"), products=products))
