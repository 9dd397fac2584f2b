"""The dense-layer and Newton-Schulz operators are not differentiated by autograd: a call whose gradient would silently be lost is refused."""
import pytest
import torch

from distributed_tensorflow_amd.ops import native as nv


def calls(device):
    f = dict(device=device)
    x, w, bias, res, dy = torch.ones(4, 6, **f), torch.ones(6, 5, **f), torch.ones(5, **f), torch.ones(4, 5, **f), torch.ones(4, 5, **f)
    return [(nv.linear, (x, w, bias), dict(residual=res)), (nv.linear_bwd, (dy, x, w), dict(pre=res, activation="silu")), (nv.newton_schulz, (x,), {})]


def tensors_of(args, kw):
    return list(args) + [t for t in kw.values() if isinstance(t, torch.Tensor)]


@pytest.mark.parametrize("which", range(3))
def test_tensors_that_require_gradients_are_refused(which):
    f, args, kw = calls("cpu")[which]
    for t in tensors_of(args, kw):
        t.requires_grad_()
        with pytest.raises(ValueError, match="no_grad"):
            f(*args, **kw)
        t.requires_grad_(False)


@pytest.mark.gpu
@pytest.mark.parametrize("which", range(3))
def test_under_no_grad_they_are_taken(which):
    f, args, kw = calls("cuda")[which]
    want = f(*args, **kw)
    for t in tensors_of(args, kw):
        t.requires_grad_()
    with torch.no_grad():
        got = f(*args, **kw)
    for a, b in zip(want if isinstance(want, tuple) else [want], got if isinstance(got, tuple) else [got]):
        assert torch.equal(a, b) and not b.requires_grad
