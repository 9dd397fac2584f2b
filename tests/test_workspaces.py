"""Workspaces that a caller brings: they are scratch memory, apart from every tensor of the call."""
import pytest
import torch

from distributed_tensorflow_amd.ops import native as nv


def test_a_workspace_that_holds_a_tensor_of_the_call_is_refused():
    buf = torch.zeros(4096)
    ws, dev = buf[1024:2048], buf.device
    apart = (buf[:1024].view(32, 32), buf[2048:].view(2, 32, 32), None)
    assert nv._workspace("linear", 256, ws, dev, apart)[2] == 4096
    for inside in (buf[1000:1032].view(4, 8), buf[2047:2063].view(4, 4), buf[1100:1104], buf[0:4096].view(4, 32, 32), buf[1536:2560].view(1, 32, 32)):
        with pytest.raises(ValueError, match="workspace"):
            nv._workspace("linear", 256, ws, dev, apart + (inside,))
    assert nv._workspace("linear", 0, None, dev, apart) == (None, 0, 0)


@pytest.mark.gpu
def test_operators_refuse_a_workspace_over_their_tensors():
    f = dict(device="cuda")
    m, k, n = 30, 4096, 64
    need = max(nv.linear_workspace(m, n, k), nv.linear_bwd_workspace(m, n, k, activation="relu"), nv.newton_schulz_workspace(m, k))
    buf = torch.zeros(need // 4 + 1024, **f)
    ws = buf[:need // 4 // 4 * 4 + 4]
    x, w, dy, bias = torch.zeros(m, k, **f), torch.zeros(k, n, **f), torch.zeros(m, n, **f), torch.zeros(n, **f)
    nv.linear(x, w, bias, workspace=ws)
    inside = {"x": buf[:m * k].view(m, k), "w": buf[:k * n].view(k, n), "dy": buf[:m * n].view(m, n), "bias": buf[:n]}
    calls = [
        lambda: nv.linear(inside["x"], w, bias, workspace=ws),
        lambda: nv.linear(x, inside["w"], bias, workspace=ws),
        lambda: nv.linear(x, w, inside["bias"], workspace=ws),
        lambda: nv.linear(x, w, bias, residual=inside["dy"], workspace=ws),
        lambda: nv.linear(x, w, bias, out=inside["dy"], workspace=ws),
        lambda: nv.linear(x, w, bias, pre=inside["dy"], workspace=ws),
        lambda: nv.linear_bwd(inside["dy"], x, w, workspace=ws),
        lambda: nv.linear_bwd(dy, inside["x"], w, workspace=ws),
        lambda: nv.linear_bwd(dy, x, inside["w"], workspace=ws),
        lambda: nv.linear_bwd(dy, x, w, pre=inside["dy"], activation="relu", workspace=ws),
        lambda: nv.linear_bwd(dy, x, w, dx=inside["x"], workspace=ws),
        lambda: nv.linear_bwd(dy, x, w, dw=inside["w"], workspace=ws),
        lambda: nv.linear_bwd(dy, x, w, db=inside["bias"], workspace=ws),
        lambda: nv.newton_schulz(inside["x"], workspace=ws),
        lambda: nv.newton_schulz(x, out=inside["x"], workspace=ws),
    ]
    for i, call in enumerate(calls):
        with pytest.raises(ValueError, match="workspace"):
            call()
            raise AssertionError(f"call {i} was accepted")
    assert not buf.any()
