"""Gradients of dense layers at the ends of the types' range: large output gradients, units that an activation shuts off."""
import pytest
import torch

from distributed_tensorflow_amd.ops import native as nv
from test_linear import U, act64, check_backward, close

F16_MAX = 65504.0


@pytest.mark.gpu
@pytest.mark.parametrize("act", ["gelu", "gelu_tanh", "silu"])
@pytest.mark.parametrize("trans_w", [False, True])
@pytest.mark.parametrize("m,k,n", [(1, 16, 24), (3, 40, 7), (20, 64, 72), (70, 33, 130), (300, 48, 264)])
def test_fp16_gradients_whose_slope_passes_one(m, k, n, trans_w, act):
    """|dy| near 65504 and slopes up to 1.13: dy act' passes fp16's range, dx and dw of small weights and inputs do not."""
    g = torch.Generator(device="cuda").manual_seed(m + n)
    pre = torch.linspace(1.2, 2.8, m * n, device="cuda").view(m, n).half()   # slopes 1.06 to 1.13
    dy = (F16_MAX * (1 - 0.02 * torch.rand(m, n, device="cuda", generator=g)) * (torch.randint(0, 2, (m, n), device="cuda", generator=g) * 2 - 1)).half()
    x = (torch.randn(m, k, device="cuda", generator=g) * 2.0 ** -8).half()
    w = (torch.randn(*((n, k) if trans_w else (k, n)), device="cuda", generator=g) * 2.0 ** -8).half()
    assert float((dy.double() * act64(pre.double(), act)[1]).abs().max()) > 1.03 * F16_MAX
    dx, dw, _ = nv.linear_bwd(dy, x, w, pre=pre, activation=act, trans_w=trans_w, db=False)
    assert bool(torch.isfinite(dx).all()) and bool(torch.isfinite(dw).all())
    check_backward(dy, x, w, pre, act, trans_w, dx, dw, None)
    base = (torch.randn(w.shape, device="cuda", generator=g)).half()
    total = base.clone()
    nv.linear_bwd(dy, x, w, pre=pre, activation=act, trans_w=trans_w, dx=False, dw=total, db=False, accumulate=True)
    check_backward(dy, x, w, pre, act, trans_w, None, total, None, base_dw=base)


@pytest.mark.gpu
@pytest.mark.parametrize("act", ["gelu", "gelu_tanh", "silu"])
def test_fp16_gradients_near_the_smallest_numbers(act):
    """Output gradients down to 2^-24. dz is rounded to multiples of 2^-23 at the least, off by 2^-24, on top of its relative rounding and the
    slope's; the sums of K products are off by (K + 4) u of their sizes, as everywhere."""
    g = torch.Generator(device="cuda").manual_seed(1)
    m, k, n = 40, 24, 56
    dy = (torch.randn(m, n, device="cuda", generator=g) * 2.0 ** -18).half()
    pre = torch.randn(m, n, device="cuda", generator=g).half()
    x = (torch.randn(m, k, device="cuda", generator=g) * 64).half()
    w = (torch.randn(k, n, device="cuda", generator=g) * 64).half()
    dx, dw, db = nv.linear_bwd(dy, x, w, pre=pre, activation=act)
    dz = dy.double() * act64(pre.double(), act)[1]
    off = dy.double().abs() * 16 * U + 2.0 ** -11 * 1.01 * dz.abs() + 2.0 ** -24
    size, w64, x64 = dz.abs() + off, w.double(), x.double()
    close(dx, dz @ w64.t(), off @ w64.abs().t() + (n + 4) * U * (size @ w64.abs().t()), torch.float16, "dx")
    close(dw, x64.t() @ dz, x64.abs().t() @ off + (m + 4) * U * (x64.abs().t() @ size), torch.float16, "dw")
    close(db, dz.sum(0), (dy.double().abs() * 16 * U).sum(0) + (m + 4) * U * dz.abs().sum(0), torch.float16, "db")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("m,k,n", [(3, 8, 5), (40, 24, 56)])
def test_relu_gradient_of_units_that_are_off(m, k, n, dtype):
    """An infinite or NaN dy at a unit that ReLU shut off leaves no trace; a NaN pre-activation stays one."""
    g = torch.Generator(device="cuda").manual_seed(2)
    dy, pre, x, w = ((torch.randn(*s, device="cuda", generator=g)).to(dtype) for s in ((m, n), (m, n), (m, k), (k, n)))
    pre[0, :3] = torch.tensor([-1.0, 0.0, -0.0])
    pre[1, 0], pre[2, 2] = float("-inf"), -3.0
    clean = dy.clone()
    clean[pre <= 0] = 0
    want = nv.linear_bwd(clean, x, w, pre=pre, activation="relu")
    dy[0, :3] = torch.tensor([float("inf"), float("-inf"), float("nan")])
    dy[1, 0] = float("nan")
    dy[2, 2] = float("inf")
    for a, b in zip(nv.linear_bwd(dy, x, w, pre=pre, activation="relu"), want):
        assert bool(torch.isfinite(a).all()) and torch.equal(a, b)
    pre[2, 1] = float("nan")
    dx, dw, db = nv.linear_bwd(dy, x, w, pre=pre, activation="relu")
    rows, cols = torch.arange(m, device="cuda") == 2, torch.arange(n, device="cuda") == 1
    assert torch.equal(dx.isnan(), rows[:, None].expand(m, k)) and torch.equal(dw.isnan(), cols.expand(k, n)) and torch.equal(db.isnan(), cols)
