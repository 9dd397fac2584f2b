"""Dense layers (ops/native.py linear, linear_bwd) against a plain 64-bit implementation.

Tolerances. u = 2^-24 is fp32's unit roundoff, r the output type's (2^-24, 2^-8 bf16, 2^-11 fp16). A sum of K
products in fp32, in any order, is off by at most (K + 1) u S with S = sum |x||w| (+ |bias|); products of 16-bit values
are exact in fp32. act' is at most 1.13 in size and the fp32 evaluation of an activation is a few u of its largest
intermediate, |z| + 1. So |y - y64| <= r |y| + 1.13 (K + 4) u S + 16 u (|z| + 1) (+ 2 u |residual|). On top of the elementwise
bound, which is loose for long K, the 2-norm of the error is held to the random-walk size, r + 2 u (sqrt(K) + 8).
fp16 results below 2^-14 are rounded to multiples of 2^-24: that much absolutely."""
import math

import pytest
import torch

from distributed_tensorflow_amd.ops import native as nv

U = 2.0 ** -24
ROUND = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
DTYPES = [torch.float32, torch.bfloat16, torch.float16]
ACTS = ["none", "relu", "gelu", "gelu_tanh", "silu"]


def act64(z, act):
    """(act(z), act'(z)) in double."""
    if act == "relu":
        return z.clamp(min=0), (z > 0).double()
    if act == "gelu":
        phi = torch.special.ndtr(z)
        return z * phi, phi + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    if act == "gelu_tanh":
        c = math.sqrt(2 / math.pi)
        t = torch.tanh(c * (z + 0.044715 * z ** 3))
        return 0.5 * z * (1 + t), 0.5 * (1 + t) + 0.5 * z * (1 - t * t) * c * (1 + 3 * 0.044715 * z * z)
    if act == "silu":
        q = torch.sigmoid(z)
        return z * q, q * (1 + z * (1 - q))
    return z, torch.ones_like(z)


def close(got, want, bound, dtype, what, norm=None):
    got, want = got.detach().double().cpu(), want.cpu()
    assert got.shape == want.shape
    tiny = 2.0 ** -24 if dtype == torch.float16 else 2.0 ** -130
    limit = ROUND[dtype] * want.abs() + bound.cpu() * 1.01 + tiny
    off = (got - want).abs()
    bad = ~(off <= limit)
    assert not bad.any(), f"{what}: {int(bad.sum())} values, worst {float((off - limit).max())} over, at {bad.nonzero()[0].tolist()}"
    if norm is not None and want.numel() > 64 and float(want.norm()) > 0:
        assert float(off.norm() / want.norm()) <= norm, f"{what}: 2-norm {float(off.norm() / want.norm())} > {norm}"


def make(m, k, n, dtype, trans_w, seed=0, pad=0, shift=0):
    """Inputs; pad > 0: views of wider buffers, shift: starting that many elements in."""
    g = torch.Generator(device="cuda").manual_seed(seed)

    def mat(r, c, scale):
        buf = torch.full((r, c + pad), float("nan"), device="cuda", dtype=dtype)
        flat = torch.full((shift + r * (c + pad),), float("nan"), device="cuda", dtype=dtype)
        view = flat[shift:].view(r, c + pad)[:, :c] if (pad or shift) else buf
        view.copy_(torch.randn(r, c, device="cuda", generator=g) * scale)
        return view

    x = mat(m, k, 1.0)
    w = mat(*((n, k) if trans_w else (k, n)), 1 / math.sqrt(max(k, 1)))
    res = mat(m, n, 1.0)
    bias = (torch.randn(n, device="cuda", generator=g) * 0.1).to(dtype)
    return x, w, bias, res


def check_forward(x, w, bias, res, act, trans_w, y, pre=None):
    dtype, k = x.dtype, x.shape[1]
    w64 = w.double().t() if trans_w else w.double()
    z = x.double() @ w64
    size = x.double().abs() @ w64.abs()
    if bias is not None:
        z, size = z + bias.double(), size + bias.double().abs()
    want, _ = act64(z, act)
    bound = 1.13 * (k + 4) * U * size + 16 * U * (z.abs() + 1)
    norm = ROUND[dtype] + 2 * U * (math.sqrt(k) + 8)
    if pre is not None:
        close(pre, z, (k + 4) * U * size, dtype, "pre", norm)
    if res is not None:
        want, bound = want + res.double(), bound + 2 * U * res.double().abs()
    close(y, want, bound, dtype, "y", 4 * norm)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("trans_w", [False, True])
@pytest.mark.parametrize("m,k,n", [(1, 1, 1), (1, 64, 8), (1, 1000, 512), (2, 33, 7), (5, 128, 130), (16, 256, 128), (17, 72, 40), (63, 31, 65),
                                   (64, 512, 64), (128, 3136, 512), (129, 127, 131), (200, 1, 300), (300, 7, 1), (257, 640, 264), (33, 2048, 48)])
def test_linear_shapes(m, k, n, trans_w, dtype):
    x, w, bias, res = make(m, k, n, dtype, trans_w)
    pre = torch.empty(m, n, device="cuda", dtype=dtype)
    y = nv.linear(x, w, bias, activation="gelu", residual=res, trans_w=trans_w, pre=pre)
    check_forward(x, w, bias, res, "gelu", trans_w, y, pre)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("trans_w", [False, True])
@pytest.mark.parametrize("m,k,n", [(4090, 200, 4088), (2000, 136, 2040), (4089, 77, 4093), (520, 8200, 136), (70, 20000, 65), (4, 8192, 1000), (1, 70000, 24),
                                   (3, 16, 9000), (8, 4096, 72)])
def test_linear_large(m, k, n, trans_w, dtype):
    """Every tile, split k, padded copies and the few-rows kernels, with edges; forward and gradients."""
    x, w, bias, res = make(m, k, n, dtype, trans_w, seed=12)
    pre = torch.empty(m, n, device="cuda", dtype=dtype)
    y = nv.linear(x, w, bias, activation="silu", residual=res, trans_w=trans_w, pre=pre)
    check_forward(x, w, bias, res, "silu", trans_w, y, pre)
    check_backward(res, x, w, pre, "silu", trans_w, *nv.linear_bwd(res, x, w, pre=pre, activation="silu", trans_w=trans_w))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("trans_w", [False, True])
@pytest.mark.parametrize("m,k,n", [(2, 1785, 283), (3, 973, 628), (5, 1024, 264), (9, 712, 3720), (23, 1000, 136), (31, 65, 260), (40, 8128, 264),
                                   (250, 2216, 304), (2, (1 << 20) + 5, 9), (70, (1 << 20) + 1, 3)])
def test_linear_few_rows_and_long_lines(m, k, n, trans_w, dtype):
    """32-row tiles, k in many parts, copies for few rows, and lines too long for a copy; forward and gradients."""
    x, w, bias, res = make(m, k, n, dtype, trans_w, seed=14)
    pre = torch.empty(m, n, device="cuda", dtype=dtype)
    y = nv.linear(x, w, bias, activation="silu", residual=res, trans_w=trans_w, pre=pre)
    check_forward(x, w, bias, res, "silu", trans_w, y, pre)
    check_backward(res, x, w, pre, "silu", trans_w, *nv.linear_bwd(res, x, w, pre=pre, activation="silu", trans_w=trans_w))


@pytest.mark.gpu
@pytest.mark.parametrize("m,k,n", [(3, 1000, 64), (20, 4096, 40), (70, 72, 136), (2, (1 << 20) + 8, 16), (2, 1 << 20, 24)])
def test_linear_workspace_covers_every_alignment(m, k, n):
    for trans_w in (False, True):
        for shift_x in (0, 1):
            for shift_w in (0, 1):
                x, _, bias, dy = make(m, k, n, torch.bfloat16, trans_w, shift=shift_x)
                _, w, _, _ = make(m, k, n, torch.bfloat16, trans_w, shift=shift_w)
                ws = torch.empty(nv.linear_workspace(m, n, k, torch.bfloat16, trans_w), device="cuda", dtype=torch.uint8)
                assert torch.equal(nv.linear(x, w, bias, trans_w=trans_w, workspace=ws), nv.linear(x, w, bias, trans_w=trans_w))
                ws = torch.empty(nv.linear_bwd_workspace(m, n, k, torch.bfloat16, trans_w), device="cuda", dtype=torch.uint8)
                for a, b in zip(nv.linear_bwd(dy, x, w, trans_w=trans_w, workspace=ws), nv.linear_bwd(dy, x, w, trans_w=trans_w)):
                    assert torch.equal(a, b)


@pytest.mark.gpu
@pytest.mark.parametrize("ld", [(1 << 22) - 8, (1 << 24) + 8, (1 << 22) + 3])
def test_linear_rows_far_apart(ld):
    """Rows whose addresses pass 2^31 and 2^32 bytes, read and written, below and above the stride that one 32-bit offset covers."""
    m, k, n = 270 if ld < 1 << 23 else 140, 72, 40
    x, w, bias, res = make(m, k, n, torch.bfloat16, False, seed=13)
    big = torch.empty(m * ld, device="cuda", dtype=torch.bfloat16)
    far = big.view(m, ld)
    xf, yf, zf = far[:, :k], far[:, 100:100 + n], far[:, 200:200 + n]
    xf.copy_(x)
    nv.linear(xf, w, bias, activation="relu", residual=res, out=yf, pre=zf)
    check_forward(x, w, bias, res, "relu", False, yf, zf)
    dyf, dxf = far[:, 300:300 + n], far[:, 400:400 + k]
    dyf.copy_(res)
    dx, dw, db = nv.linear_bwd(dyf, xf, w, pre=zf, activation="relu", dx=dxf)
    check_backward(res, x, w, zf, "relu", False, dxf, dw, db)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("act", ACTS)
def test_linear_activations(act, dtype):
    x, w, bias, _ = make(40, 96, 56, dtype, False, seed=1)
    y = nv.linear(x * 3, w, bias, activation=act)
    check_forward(x * 3, w, bias, None, act, False, y)
    check_forward(x, w, None, None, act, False, nv.linear(x, w, activation=act))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("pad,shift", [(8, 0), (8, 8), (3, 0), (1, 1), (0, 1), (5, 3)])
@pytest.mark.parametrize("m,k,n", [(20, 64, 24), (1, 200, 136), (150, 136, 144), (9, 129, 33)])
def test_linear_strides_and_alignment(m, k, n, pad, shift, dtype):
    """Views whose surroundings are NaN: nothing outside the matrices is used, and nothing outside the output is written."""
    for trans_w in (False, True):
        x, w, bias, res = make(m, k, n, dtype, trans_w, seed=2, pad=pad, shift=shift)
        store = torch.full((shift + m * (n + pad) + 7,), 5.0, device="cuda", dtype=dtype)
        y = store[shift:shift + m * (n + pad)].view(m, n + pad)[:, :n]
        pstore = store.clone()
        pre = pstore[shift:shift + m * (n + pad)].view(m, n + pad)[:, :n]
        assert nv.linear(x, w, bias, activation="silu", residual=res, trans_w=trans_w, out=y, pre=pre) is y
        check_forward(x, w, bias, res, "silu", trans_w, y, pre)
        for s in (store, pstore):
            rest = torch.ones_like(s, dtype=torch.bool)
            rest[shift:shift + m * (n + pad)].view(m, n + pad)[:, :n] = False
            assert bool((s[rest] == 5).all())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_linear_in_place_residual_and_empty_sizes(dtype):
    x, w, bias, res = make(70, 48, 50, dtype, False, seed=3)
    keep = res.clone()
    y = nv.linear(x, w, bias, activation="relu", residual=res, out=res)
    assert y is res
    check_forward(x, w, bias, keep, "relu", False, y)
    e = torch.empty
    kw = dict(device="cuda", dtype=dtype)
    assert nv.linear(e(0, 8, **kw), e(8, 4, **kw)).shape == (0, 4)
    assert nv.linear(e(3, 8, **kw), e(8, 0, **kw)).shape == (3, 0)
    b = torch.tensor([1.0, -2.0], **kw)
    assert torch.equal(nv.linear(e(3, 0, **kw), e(0, 2, **kw), b, activation="relu"), torch.tensor([[1.0, 0.0]] * 3, **kw))
    dx, dw, db = nv.linear_bwd(e(0, 4, **kw), e(0, 8, **kw), torch.ones(8, 4, **kw))
    assert dx.shape == (0, 8) and not dw.any() and not db.any() and dw.shape == (8, 4)
    dx, dw, db = nv.linear_bwd(e(3, 0, **kw), torch.ones(3, 8, **kw), e(8, 0, **kw))
    assert dx.shape == (3, 8) and not dx.any() and dw.shape == (8, 0) and db.shape == (0,)
    dw, db = torch.ones(8, 4, **kw), torch.ones(4, **kw)
    nv.linear_bwd(e(0, 4, **kw), e(0, 8, **kw), torch.ones(8, 4, **kw), dx=False, dw=dw, db=db, accumulate=True)
    assert bool((dw == 1).all()) and bool((db == 1).all())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m", [3, 40, 200])
def test_linear_infinities_and_nan_stay_in_their_rows(m, dtype):
    x, w, bias, _ = make(m, 80, 48, dtype, False, seed=4)
    w.abs_()
    x.abs_()
    clean = nv.linear(x, w, bias, activation="relu")
    x[1, 7] = float("inf")
    x[2, 5] = float("nan")
    y = nv.linear(x, w, bias, activation="relu")
    assert bool((y[1] == float("inf")).all()) and bool(y[2].isnan().all())
    keep = [i for i in range(m) if i not in (1, 2)]
    assert torch.equal(y[keep], clean[keep])


def check_backward(dy, x, w, pre, act, trans_w, dx, dw, db, base_dw=None, base_db=None):
    dtype, (m, n), k = dy.dtype, dy.shape, x.shape[1]
    _, grad = act64(pre.double() if pre is not None else torch.zeros(m, n, dtype=torch.float64, device=dy.device), act)
    dz = dy.double() * grad
    # act' is evaluated in fp32: off by a few u of terms no larger than 1 + z^2 phi(z) ... <= 2; then dz is rounded to the type
    dzo = dy.double().abs() * 16 * U + (ROUND[dtype] * 1.01 if act not in ("none", "relu") else 0) * dz.abs()
    if dtype == torch.float16 and act not in ("none", "relu"):
        dzo = dzo + 2.0 ** -24
    w64, x64 = (w.double().t() if trans_w else w.double()), x.double()
    adz = dz.abs() + dzo
    norm = 2 * ROUND[dtype] + 2 * U
    if dx is not None:
        close(dx, dz @ w64.t(), dzo @ w64.abs().t() + (n + 4) * U * (adz @ w64.abs().t()), dtype, "dx", norm + 2 * U * (math.sqrt(n) + 8))
    if dw is not None:
        want = x64.t() @ dz
        bound = x64.abs().t() @ dzo + (m + 4) * U * (x64.abs().t() @ adz)
        want, bound = (want.t(), bound.t()) if trans_w else (want, bound)
        if base_dw is not None:
            want, bound = want + base_dw.double(), bound + 2 * U * base_dw.double().abs()
        close(dw, want, bound, dtype, "dw", norm + 2 * U * (math.sqrt(m) + 8))
    if db is not None:
        want = dz.sum(0)
        bound = (dy.double().abs() * 16 * U).sum(0) + (m + 4) * U * dz.abs().sum(0)
        if base_db is not None:
            want, bound = want + base_db.double(), bound + 2 * U * base_db.double().abs()
        close(db, want, bound, dtype, "db")


def make_backward(m, k, n, dtype, trans_w, seed=0, pad=0, shift=0):
    x, w, _, dy = make(m, k, n, dtype, trans_w, seed, pad, shift)
    pre = (torch.randn(m, n + pad, device="cuda", generator=torch.Generator(device="cuda").manual_seed(seed + 9)) * 1.5).to(dtype)[:, :n]
    return dy, x, w, pre


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("trans_w", [False, True])
@pytest.mark.parametrize("m,k,n", [(1, 1, 1), (1, 512, 256), (3, 65, 30), (16, 64, 64), (20, 9, 300), (64, 100, 10), (128, 3136, 512), (130, 264, 136),
                                   (1000, 48, 40), (700, 31, 33)])
def test_linear_bwd_shapes(m, k, n, trans_w, dtype):
    dy, x, w, pre = make_backward(m, k, n, dtype, trans_w)
    check_backward(dy, x, w, pre, "silu", trans_w, *nv.linear_bwd(dy, x, w, pre=pre, activation="silu", trans_w=trans_w))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("act", ACTS)
def test_linear_bwd_activations_and_choices(act, dtype):
    dy, x, w, pre = make_backward(50, 72, 40, dtype, False, seed=5)
    pre[0, :4] = torch.tensor([0.0, -0.0, 30.0, -30.0])
    p = None if act == "none" else pre
    full = nv.linear_bwd(dy, x, w, pre=p, activation=act)
    check_backward(dy, x, w, pre, act, False, *full)
    for choice in ((True, False, False), (False, True, False), (False, False, True), (True, None, True)):
        part = nv.linear_bwd(dy, x, w, pre=p, activation=act, dx=choice[0], dw=choice[1], db=choice[2])
        for c, a, b in zip(choice, part, full):
            assert (a is None) if not c else torch.equal(a, b)
    assert nv.linear_bwd(dy, x, w, pre=p, activation=act, dx=False, dw=False, db=False) == (None, None, None)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("pad,shift", [(8, 8), (3, 1)])
def test_linear_bwd_strided_accumulating(pad, shift, dtype):
    for trans_w in (False, True):
        dy, x, w, pre = make_backward(45, 56, 24, dtype, trans_w, seed=6, pad=pad, shift=shift)
        g = torch.Generator(device="cuda").manual_seed(8)
        dw0 = torch.randn(w.shape[0], w.shape[1] + pad, device="cuda", generator=g).to(dtype)
        db0 = torch.randn(24, device="cuda", generator=g).to(dtype)
        dw, db, dx = dw0.clone()[:, :w.shape[1]], db0.clone(), torch.zeros(45, 56 + pad, device="cuda", dtype=dtype)[:, :56]
        nv.linear_bwd(dy, x, w, pre=pre, activation="gelu_tanh", trans_w=trans_w, dx=dx, dw=dw, db=db, accumulate=True)
        check_backward(dy, x, w, pre, "gelu_tanh", trans_w, dx, dw, db, dw0[:, :w.shape[1]], db0)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("act", ACTS[1:])
def test_linear_bwd_slopes_far_out(act, dtype):
    """Pre-activations far from zero, up to infinity: the slope is 0 or 1 to the last bit, and NaN stays NaN."""
    far = [300.0, 65504.0, 1e20, 3e38, float("inf")]
    pre = torch.tensor([far, [-v for v in far]], dtype=torch.float64).to(dtype).cuda()
    dy = torch.full((2, 5), 2.0, dtype=dtype, device="cuda")
    eye = torch.eye(5, dtype=dtype, device="cuda")
    x = torch.ones(2, 3, dtype=dtype, device="cuda")
    dx, dw, db = nv.linear_bwd(dy, x, eye[:3].contiguous(), pre=pre, activation=act)
    assert torch.equal(dx, torch.tensor([[2.0] * 3, [0.0] * 3], dtype=dtype, device="cuda"))
    assert torch.equal(db, torch.full((5,), 2.0, dtype=dtype, device="cuda")) and torch.equal(dw, torch.full((3, 5), 2.0, dtype=dtype, device="cuda"))
    if act != "relu":
        pre[0, 1] = float("nan")
        db = nv.linear_bwd(dy, x, eye[:3].contiguous(), pre=pre, activation=act)[2]
        assert db.isnan().tolist() == [False, True, False, False, False]


@pytest.mark.gpu
def test_linear_gradients_against_differences():
    """Directional derivatives of sum(c * y) by central differences in 64 bits against the fp32 kernels' gradients."""
    m, k, n = 12, 20, 9
    x, w, bias, c = make(m, k, n, torch.float32, False, seed=11)
    for act in ("gelu", "gelu_tanh", "silu"):
        pre = torch.empty(m, n, device="cuda")
        nv.linear(x, w, bias, activation=act, pre=pre)
        dx, dw, db = nv.linear_bwd(c, x, w, pre=pre, activation=act)

        def loss(xx, ww, bb):
            return float((c.double() * act64(xx @ ww + bb, act)[0]).sum())

        g = torch.Generator(device="cuda").manual_seed(3)
        for grad, pick in ((dx, 0), (dw, 1), (db, 2)):
            at = [x.double(), w.double(), bias.double()]
            d = torch.randn(grad.shape, device="cuda", generator=g).double()
            h = 1e-4
            lo, hi = list(at), list(at)
            lo[pick], hi[pick] = at[pick] - h * d, at[pick] + h * d
            want = (loss(*hi) - loss(*lo)) / (2 * h)
            # the differences are off by h^2/6 times a third derivative of sum |c||d|..., below 1e-6 here; the gradient by 1e-5 of its size
            assert abs(float((grad.double() * d).sum()) - want) <= 1e-5 * float((grad.double() * d).abs().sum()) + 1e-4


@pytest.mark.gpu
def test_linear_layers_together_in_a_graph_replay():
    """A two-layer network's forward and backward pass, captured once and replayed on new inputs between eager calls."""
    g = torch.Generator(device="cuda").manual_seed(1)
    kw = dict(device="cuda", dtype=torch.bfloat16)
    x = torch.randn(48, 136, device="cuda", generator=g).bfloat16()
    w1 = (torch.randn(136, 520, device="cuda", generator=g) / 12).bfloat16()
    w2 = (torch.randn(520, 136, device="cuda", generator=g) / 23).bfloat16()
    b1, b2, dy = torch.zeros(520, **kw), torch.ones(136, **kw), torch.randn(48, 136, device="cuda", generator=g).bfloat16()

    def both():
        pre = torch.empty(48, 520, **kw)
        h = nv.linear(x, w1, b1, activation="gelu", pre=pre)
        y = nv.linear(h, w2, b2, residual=x)
        dh, dw2, db2 = nv.linear_bwd(dy, h, w2)
        dx, dw1, db1 = nv.linear_bwd(dh, x, w1, pre=pre, activation="gelu")
        return [y, dx, dw1, db1, dw2, db2]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        both()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            held = both()
    torch.cuda.current_stream().wait_stream(side)
    for seed in range(3):
        x.copy_(torch.randn(48, 136, device="cuda", generator=torch.Generator(device="cuda").manual_seed(seed + 20)))
        want = both()
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(held, want):
            assert torch.equal(a, b)   # every sum has a fixed order


@pytest.mark.gpu
def test_linear_on_another_stream_and_recorded():
    x, w, bias, _ = make(30, 4096, 64, torch.float32, False, seed=7)
    want = nv.linear(x, w, bias, activation="relu")
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        got = nv.linear(x, w, bias, activation="relu")
    s.synchronize()
    assert torch.equal(got, want)
    need = nv.linear_workspace(30, 64, 4096)
    ws, out = torch.empty(need + 16, device="cuda", dtype=torch.uint8), torch.zeros(30, 64, device="cuda")
    prog = nv.hip().Program()
    prog.begin_record()
    try:
        if need:
            with pytest.raises(ValueError, match="workspace"):
                nv.linear(x, w, bias, activation="relu", out=out)
        nv.linear(x, w, bias, activation="relu", out=out, workspace=ws)
    finally:
        prog.end_record()
    assert not out.any()
    prog.run(torch.cuda.current_stream().cuda_stream, -1)
    torch.cuda.synchronize()
    assert torch.equal(out, want)


def test_linear_refuses_bad_arguments():
    f = torch.zeros
    x, w = f(4, 6), f(6, 5)
    bad = [
        lambda: nv.linear(f(4), w),
        lambda: nv.linear(x, f(5, 6)),
        lambda: nv.linear(x, w, trans_w=True),
        lambda: nv.linear(x, w.double()),
        lambda: nv.linear(x.double(), w.double()),
        lambda: nv.linear(x.int(), w.int()),
        lambda: nv.linear(x, w, f(6)),
        lambda: nv.linear(x, w, f(5).bfloat16()),
        lambda: nv.linear(x, w, f(10)[::2]),
        lambda: nv.linear(x, w, activation="tanh"),
        lambda: nv.linear(x, w, residual=f(4, 6)),
        lambda: nv.linear(x, w, residual=f(4, 5).half()),
        lambda: nv.linear(x, w, out=f(5, 4)),
        lambda: nv.linear(x, w, out=f(5, 4).t()),
        lambda: nv.linear(x, w, out=f(1, 5).expand(4, 5)),
        lambda: nv.linear(x, w, pre=f(4, 4)),
        lambda: nv.linear(f(6, 4).t(), w),
        lambda: nv.linear(x, f(6, 6), out=x),
        lambda: nv.linear_bwd(f(4, 5), f(3, 6), w),
        lambda: nv.linear_bwd(f(4, 5), x, f(5, 6)),
        lambda: nv.linear_bwd(f(4, 5), x, w, activation="relu"),
        lambda: nv.linear_bwd(f(4, 5), x, w, activation="relu", pre=f(5, 4)),
        lambda: nv.linear_bwd(f(4, 5), x, w, activation="swish"),
        lambda: nv.linear_bwd(f(4, 5), x, w, accumulate=True),
        lambda: nv.linear_bwd(f(4, 5), x, w, dw=f(5, 6)),
        lambda: nv.linear_bwd(f(4, 5), x, w, db=f(6)),
        lambda: nv.linear_bwd(f(4, 5), x, w, dx=x),
        lambda: nv.linear_bwd(f(4, 5).bfloat16(), x, w),
    ]
    for i, call in enumerate(bad):
        with pytest.raises(ValueError):
            call()
            raise AssertionError(f"call {i} was accepted")
    out = f(4, 5)
    with pytest.raises(ValueError):
        nv.linear(x, w, residual=f(5 * 5)[2:22].view(4, 5), out=out, pre=out)
    wide = f(4, 20)
    assert not nv._overlap(wide[:, :6], wide[:, 6:11]) and not nv._overlap(wide[:, 6:11], wide[:, :6]) and not nv._overlap(wide[:, 15:], wide[1:, :15])
    assert nv._overlap(wide[:, :7], wide[:, 6:11]) and nv._overlap(wide[:, 2:4], wide[:, :20]) and nv._overlap(wide[1:, :6], wide[:, :6])
    with pytest.raises(ValueError):
        nv.linear(wide[:, :6], w, out=wide[:, 5:10])
    buf = f(40)
    with pytest.raises(ValueError):
        nv.linear(x, w, residual=buf[0:20].view(4, 5), out=buf[10:30].view(4, 5))


def test_linear_workspace_refusals():
    if nv._hip is None:
        pytest.skip("extension not built")
    dev = torch.device("cpu")
    for m, n, k in ((0, 4, 8), (3, 0, 8), (3, 4, 0), (0, 0, 0), (1, 1, 1), (8192, 7, 70000)):
        assert nv.linear_workspace(m, n, k) >= 0 and nv.linear_bwd_workspace(m, n, k, activation="silu") >= 0
    ok = torch.empty(64, dtype=torch.uint8)
    assert nv._workspace("linear", 0, None, dev) == (None, 0, 0)
    assert nv._workspace("linear", 32, ok, dev)[2] == 64
    with pytest.raises(ValueError):
        nv._workspace("linear", 65, ok, dev)
    with pytest.raises(ValueError):
        nv._workspace("linear", 8, ok[1:], dev)
    with pytest.raises(ValueError):
        nv._workspace("linear", 8, ok[::2], dev)


def test_linear_refuses_sizes_past_its_indices():
    """Dimensions that a tile's 32-bit indices or a launch's threads could not count: refused when the workspace is asked for."""
    if nv._hip is None:
        pytest.skip("extension not built")
    top = 2 ** 31
    for m, n, k in ((top - 1, 1, 1), (1, top - 1, 1), (1, 1, top - 1), (top - 65536, 512, 8), (512, top - 65536, 8)):
        with pytest.raises(RuntimeError, match="dimension|too many tiles"):
            nv.linear_workspace(m, n, k)
    with pytest.raises(RuntimeError, match="too many tiles"):   # 16 columns a workgroup of 1024 threads
        nv.linear_workspace(1, 2 ** 27, 8, torch.bfloat16, trans_w=True)
    with pytest.raises(RuntimeError, match="too many tiles"):   # column sums, 64 columns a workgroup of 256
        nv.linear_bwd_workspace(1, 2 ** 30, 1)
    with pytest.raises(RuntimeError, match="dimension"):
        nv.linear_bwd_workspace(1, top - 1, 1)
