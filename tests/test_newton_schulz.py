"""Newton-Schulz orthogonalisation and the optimizer built on it, against a 64-bit statement of the formulas.

Tolerance of a result, in the Frobenius norm: a step's products leave a relative error eta in X, and a later step magnifies it
by at most L = max |d/ds (a s + b s^3 + c s^5)| over the singular values that occur (the Lipschitz bound of an odd matrix
polynomial), so the error is at most sum_k L^(n-k) eta |X_k|, with the |X_k| of the 64-bit iteration. eta counts
the pairs (22 bits: X, P and A rounded to 2^-22 each, the dropped l l products 2^-22; doubled for A's two uses) and the random walk of
fp32 sums of r and c terms: eta = 8 * 2^-22 + 2^-23 (sqrt(r) + sqrt(c)). The output adds its own rounding."""
import math

import numpy as np
import pytest
import torch

from distributed_tensorflow_amd.models.lenet import lenet_param_specs
from distributed_tensorflow_amd.models.resnet import resnet_param_specs
from distributed_tensorflow_amd.ops import native as nv
from distributed_tensorflow_amd.ops import reference as ref
from distributed_tensorflow_amd.optim import FlatMuon
from distributed_tensorflow_amd.runtime.arena import ParamArena, ParamSpec

ROUND = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def ns64(g, steps=5, coeffs=ref.NS_COEFFS, eps=1e-7):
    """(result, error bound in the Frobenius norm before the output's rounding)"""
    per = [coeffs] * steps if not isinstance(coeffs[0], (tuple, list)) else list(coeffs)
    x = g.double()
    x = x if x.numel() > 1 << 20 else x.cpu()
    tall = x.shape[0] > x.shape[1]
    x = x.t() if tall else x
    r, c = x.shape
    x = x / (x.norm() + eps)
    eta = 8 * 2.0 ** -22 + 2.0 ** -23 * (math.sqrt(r) + math.sqrt(c))
    err, top = eta * float(x.norm()), 1.001
    for a, b, cc in per:
        s = torch.linspace(0, top, 2001, dtype=torch.float64)
        lip = float((a + 3 * b * s ** 2 + 5 * cc * s ** 4).abs().max())
        lip = max(lip, float((a + b * s ** 2 + cc * s ** 4).abs().max()))
        top = 1.001 * float((s * (a + b * s ** 2 + cc * s ** 4)).abs().max())
        m = x @ x.t()
        x = a * x + (b * m + cc * m @ m) @ x
        err = lip * err + eta * float(x.norm())
    return (x.t() if tall else x).cpu(), err


def check(out, g, steps=5, coeffs=ref.NS_COEFFS, eps=1e-7):
    want, err = ns64(g, steps, coeffs, eps)
    tiny = 2.0 ** -25 * math.sqrt(want.numel()) if out.dtype == torch.float16 else 0.0
    got = out.double().cpu()
    assert bool(torch.isfinite(got).all())
    off, limit = float((got - want).norm()), err + ROUND[out.dtype] * float(want.norm()) + tiny
    assert off <= limit, f"{tuple(g.shape)}: off by {off}, at most {limit} (result {float(want.norm())})"


def gradient(m, n, seed=0, scale=1e-3, noise=0.05, batch=None):
    g = torch.Generator().manual_seed(seed)
    b = () if batch is None else (batch,)
    k = min(16, m, n)
    fall = 0.5 ** torch.linspace(0, 6, k)
    x = (torch.randn(*b, m, k, generator=g) * fall) @ torch.randn(*b, k, n, generator=g) / math.sqrt(k) + noise * torch.randn(*b, m, n, generator=g)
    return x * scale


SHAPES = [(1, 1), (1, 9), (9, 1), (2, 3), (10, 64), (64, 10), (16, 16), (31, 33), (33, 31), (27, 16), (144, 16), (32, 288), (64, 64), (65, 64),
          (96, 160), (128, 128), (130, 70), (300, 520), (800, 64), (257, 1030), (512, 512), (520, 264)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m,n", SHAPES)
def test_newton_schulz_shapes(m, n, dtype):
    g = gradient(m, n, seed=m * 7 + n, scale=1.0 if dtype == torch.float16 else 1e-3).to(dtype).cuda()
    keep = g.clone()
    out = nv.newton_schulz(g)
    assert out.shape == g.shape and out.dtype == dtype and torch.equal(g, keep)
    check(out, g)


@pytest.mark.gpu
@pytest.mark.parametrize("m,n,dtype", [(1500, 2600, torch.float32), (2600, 1111, torch.float16), (2048, 2050, torch.float32), (4090, 4000, torch.float32),
                                       (1024, 4096, torch.bfloat16), (130, 9000, torch.float32), (9000, 100, torch.bfloat16), (3, 40000, torch.float32),
                                       (769, 64, torch.float32), (768, 64, torch.float32), (32, 1024, torch.float32), (1025, 32, torch.float32)])
def test_newton_schulz_large(m, n, dtype):
    """The larger tiles, the split X X^T, and both sides of the border of the one-workgroup kernel."""
    g = gradient(m, n, seed=3, scale=1.0).to(dtype).cuda()
    check(nv.newton_schulz(g), g)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("m,n", [(1, 2048), (9, 1486), (2000, 9), (16, 2048), (1025, 16), (16, 2049), (17, 1100)])
def test_newton_schulz_few_long_rows(m, n, dtype):
    g = gradient(m, n, seed=5, scale=1.0).to(dtype).cuda()
    check(nv.newton_schulz(g), g)


@pytest.mark.gpu
@pytest.mark.parametrize("batch", [1, 2, 6, 40])
@pytest.mark.parametrize("m,n", [(576, 64), (48, 40), (20, 200)])
def test_newton_schulz_batches(m, n, batch):
    g = gradient(m, n, seed=batch, batch=batch).cuda()
    g[0] *= 1e4
    out = nv.newton_schulz(g)
    for i in range(batch):
        check(out[i], g[i])
        assert torch.equal(out[i], nv.newton_schulz(g[i])) or batch > 1   # the tiles may differ with the batch, the formula does not
    again = nv.newton_schulz(g)
    assert torch.equal(out, again)   # fixed orders


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_newton_schulz_strided_and_in_place(dtype):
    for m, n in ((40, 24), (24, 41), (70, 70)):
        src = gradient(m, n, batch=3, scale=1.0).to(dtype).cuda()
        wide = torch.full((3, m + 2, n + 5), float("nan"), device="cuda", dtype=dtype)
        g = wide[:, 1:m + 1, 3:n + 3]
        g.copy_(src)
        store = torch.full((3, m + 1, n + 3), 7.0, device="cuda", dtype=dtype)
        out = store[:, :m, 1:n + 1]
        assert nv.newton_schulz(g, out=out) is out
        for i in range(3):
            check(out[i], src[i])
        mask = torch.ones_like(store, dtype=torch.bool)
        mask[:, :m, 1:n + 1] = False
        assert bool((store[mask] == 7).all())
        want = out.clone()
        nv.newton_schulz(g, out=g)
        assert torch.equal(g, want) and bool(wide[:, 0].isnan().all()) and bool(wide[:, :, n + 3:].isnan().all())
        # batches of stride zero (one matrix read several times) and transposed batches of rows
        same = nv.newton_schulz(src[:1].expand(4, m, n))
        assert all(torch.equal(same[0], same[i]) for i in range(4))
        inter = src.permute(1, 0, 2).contiguous().permute(1, 0, 2)
        assert torch.equal(nv.newton_schulz(inter), nv.newton_schulz(src))


@pytest.mark.gpu
@pytest.mark.parametrize("scale", [1e18, 1e3, 1e-6, 1e-9, 1e-12, 1e-20, 1e-34, 1e-38])
def test_newton_schulz_norms_far_from_one(scale):
    """Squares leave fp32's range on both sides; far below eps the result is the linear part, far below one."""
    for m, n in ((40, 72), (96, 64), (130, 200), (300, 140)):
        g = (gradient(m, n, seed=4, scale=1.0) * scale).cuda()
        check(nv.newton_schulz(g), g)


@pytest.mark.gpu
def test_newton_schulz_special_matrices():
    zero = torch.zeros(40, 30, device="cuda")
    assert not nv.newton_schulz(zero).any()
    eye = torch.eye(64, device="cuda")
    check(nv.newton_schulz(eye * 3), eye * 3)
    rank1 = torch.outer(torch.arange(1.0, 51.0), torch.linspace(-1, 1, 90)).cuda()
    check(nv.newton_schulz(rank1), rank1)
    spike = torch.full((60, 60), 1e-5, device="cuda")
    spike[3, 4] = 1e4
    check(nv.newton_schulz(spike), spike)
    q = torch.linalg.qr(torch.randn(200, 96, generator=torch.Generator().manual_seed(1)))[0].contiguous().cuda()
    s = torch.linalg.svdvals(nv.newton_schulz(q).double().cpu())
    assert float(s.min()) > 0.6 and float(s.max()) < 1.25
    batch = gradient(50, 70, batch=3).cuda()
    clean = nv.newton_schulz(batch)
    for bad in (float("nan"), float("inf"), float("-inf")):
        b = batch.clone()
        b[1, 5, 6] = bad
        out = nv.newton_schulz(b)
        assert bool(out[1].isnan().all()) and torch.equal(out[0], clean[0]) and torch.equal(out[2], clean[2])


@pytest.mark.gpu
@pytest.mark.parametrize("steps,coeffs,eps", [(1, ref.NS_COEFFS, 1e-7), (2, ref.NS_COEFFS, 1e-3), (12, (1.5, -0.5, 0.0), 1e-7), (6, (2.0, -1.5, 0.5), 1e-7),
                                              (2, ((3.4445, -4.775, 2.0315), (1.5, -0.5, 0.0)), 1e-30), (3, (1.0, 0.0, 0.0), 1e-7)])
def test_newton_schulz_other_sequences(steps, coeffs, eps):
    for m, n in ((33, 80), (80, 33)):
        g = gradient(m, n, seed=6).cuda()
        check(nv.newton_schulz(g, steps=steps, coeffs=coeffs, eps=eps), g, steps, coeffs, eps)


@pytest.mark.gpu
def test_newton_schulz_empty():
    for shape in ((0, 4), (4, 0), (0, 3, 3), (2, 0, 3), (2, 3, 0)):
        assert nv.newton_schulz(torch.empty(shape, device="cuda")).shape == shape


@pytest.mark.gpu
def test_newton_schulz_graph_replay_and_stream():
    g = gradient(100, 140).cuda()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        nv.newton_schulz(g)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            held = nv.newton_schulz(g)
    torch.cuda.current_stream().wait_stream(s)
    for seed in range(3):
        g.copy_(gradient(100, 140, seed=30 + seed, scale=10.0 ** (-seed * 5)).cuda())
        want = nv.newton_schulz(g)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(held, want)


def test_newton_schulz_refuses_bad_arguments():
    f = torch.zeros
    for call in (lambda: nv.newton_schulz(f(4)), lambda: nv.newton_schulz(f(2, 2, 2, 2)), lambda: nv.newton_schulz(f(4, 4), steps=0),
                 lambda: nv.newton_schulz(f(4, 4), steps=17), lambda: nv.newton_schulz(f(4, 4), eps=0.0), lambda: nv.newton_schulz(f(4, 4), eps=-1.0),
                 lambda: nv.newton_schulz(f(4, 4), eps=float("nan")), lambda: nv.newton_schulz(f(4, 4), coeffs=(1.0, 2.0)),
                 lambda: nv.newton_schulz(f(4, 4), coeffs=((1.0, 0.0, 0.0),)), lambda: nv.newton_schulz(f(4, 4), coeffs=(3.0, 0.0, 0.0)),
                 lambda: nv.newton_schulz(f(4, 4), coeffs=(float("inf"), 0.0, 0.0)), lambda: nv.newton_schulz(f(4, 6), out=f(6, 4)),
                 lambda: nv.newton_schulz(f(4, 6), out=f(4, 6).half()), lambda: nv.newton_schulz(f(6, 4).t()),
                 lambda: nv.newton_schulz(f(4, 4).double()), lambda: nv.newton_schulz(f(4, 4).int()),
                 lambda: nv.newton_schulz(f(3, 4, 4), out=f(1, 4, 4).expand(3, 4, 4)), lambda: nv.newton_schulz(f(4, 6), out=f(1, 6).expand(4, 6))):
        with pytest.raises(ValueError):
            call()


def test_newton_schulz_refuses_sizes_past_its_indices():
    """32-bit offsets inside a tile: rows x 4-byte elements of up to 256 rows have to stay within 2^32."""
    if nv._hip is None:
        pytest.skip("extension not built")
    assert nv.newton_schulz_workspace(32, 2 ** 25) > 0 and nv.newton_schulz_workspace(2 ** 22, 256) > 0
    for m, n in ((65, 2 ** 24), (2 ** 24, 65), (32, 2 ** 25 + 1), (256, 2 ** 22 + 1), (1, 2 ** 30 + 1), (2 ** 31 - 1, 1)):
        with pytest.raises(RuntimeError, match="too long|dimension"):
            nv.newton_schulz_workspace(m, n)


def test_growth_bounds_the_sequence():
    """The accepted sequences keep singular values within 3.8 (brute force over a fine grid)."""
    for coeffs in (ref.NS_COEFFS, (1.5, -0.5, 0.0), (2.0, -1.5, 0.5), (4.0848, -6.8946, 2.927)):
        flat, growth = nv._ns_steps(coeffs, 8)
        s = np.linspace(0, 1, 20001)
        for a, b, c in np.asarray(flat).reshape(-1, 3):
            assert np.abs(a + b * s ** 2 + c * s ** 4).max() <= growth
            s = np.abs(s * (a + b * s ** 2 + c * s ** 4))
            assert s.max() <= 3.8


# ----------------------------------------------------------------------------- the optimizer
def _arena(specs, device="cpu"):
    a = ParamArena(specs, device, FlatMuon.slots)
    a.initialize(1)
    return a


def muon64(state, specs, offsets, grads, t, lr, gs, vlr, mu=0.95, nesterov=True, wd=0.0, named=None, steps=5):
    """One step in 64 bits over flat buffers; returns the bound on the matrices' error."""
    p, m, v = state
    g = grads.double() * gs
    lr_t = vlr * math.sqrt(1 - 0.999 ** t) / (1 - 0.9 ** t)
    bound = torch.zeros_like(p)
    for s in specs:
        at = slice(offsets[s.name], offsets[s.name] + s.numel)
        if len(s.shape) >= 2 and (named is None or s.name in named):
            rows, cols = s.numel // s.shape[-1], s.shape[-1]
            m[at] = mu * m[at] + g[at]
            u = g[at] + mu * m[at] if nesterov else m[at]
            o, err = ns64(u.view(rows, cols), steps)
            step = lr * math.sqrt(max(1.0, cols / rows))
            p[at] = (1 - lr * wd) * p[at] - step * o.reshape(-1)
            bound[at] = step * err
        else:
            m[at] = 0.9 * m[at] + 0.1 * g[at]
            v[at] = 0.999 * v[at] + 0.001 * g[at] ** 2
            p[at] = p[at] - lr_t * m[at] / (v[at].sqrt() + 1e-8)
    return bound


def run_steps(arena, specs, opt, n, **kw):
    offs = arena.offsets
    state = [t.double().cpu() for t in (arena.params, arena.slots["m"], arena.slots["v"])]
    total_bound = torch.zeros_like(state[0])
    for t in range(1, n + 1):
        gen = torch.Generator().manual_seed(100 + t)
        grad = torch.zeros(arena.total)
        for s in specs:
            at = slice(offs[s.name], offs[s.name] + s.numel)
            if len(s.shape) >= 2:
                grad[at] = gradient(s.numel // s.shape[-1], s.shape[-1], seed=t * 1000 + offs[s.name] % 997).reshape(-1)
            else:
                grad[at] = 1e-3 * torch.randn(s.numel, generator=gen)
        arena.grads.copy_(grad)
        opt.step(0.02, grad_scale=0.5, vector_lr=1e-3)
        total_bound += muon64(state, specs, offs, grad, t, 0.02, 0.5, 1e-3, **kw)
    for s in specs:
        at = slice(offs[s.name], offs[s.name] + s.numel)
        got, want = arena.params[at].double().cpu(), state[0][at]
        # the matrices' bound is on their norm; momentum and the update add a few roundings of p and of lr * o
        limit = float(total_bound[at].max()) * 1.0 + 4 * n * 2.0 ** -24 * float(want.norm()) + n * 2.0 ** -22 * 0.05 * math.sqrt(s.numel)
        assert float((got - want).norm()) <= limit, (s.name, float((got - want).norm()), limit)
        for slot, w in (("m", state[1]), ("v", state[2])):
            assert torch.allclose(arena.slots[slot][at].double().cpu(), w[at], rtol=4 * n * 2.0 ** -23, atol=1e-9 if slot == "m" else 1e-14)
    assert opt.steps == n


ODD_SPECS = [ParamSpec("a", (5, 7), "trunc_normal"), ParamSpec("b", (13,), "ones"), ParamSpec("c", (3, 3, 3, 70), "trunc_normal"),
             ParamSpec("d", (1, 40), "trunc_normal"), ParamSpec("e", (2500,), "ones"), ParamSpec("f", (130, 1), "trunc_normal"),
             ParamSpec("g", (200, 90), "trunc_normal"), ParamSpec("h", (90, 200), "trunc_normal"), ParamSpec("i", (), "ones")]


@pytest.mark.parametrize("nesterov,wd", [(True, 0.0), (False, 0.1)])
def test_flat_muon_cpu(nesterov, wd):
    a = _arena(ODD_SPECS)
    run_steps(a, ODD_SPECS, FlatMuon(a, nesterov=nesterov, weight_decay=wd), 2, nesterov=nesterov, wd=wd)


@pytest.mark.gpu
@pytest.mark.parametrize("specs,nesterov,wd", [(ODD_SPECS, True, 0.0), (ODD_SPECS, False, 0.1), (lenet_param_specs(), True, 0.01), (resnet_param_specs(2), True, 0.0)])
def test_flat_muon_gpu(specs, nesterov, wd):
    a = _arena(specs, "cuda")
    run_steps(a, specs, FlatMuon(a, nesterov=nesterov, weight_decay=wd), 3, nesterov=nesterov, wd=wd)
    pad = torch.ones(a.capacity, dtype=torch.bool)
    for s in specs:
        pad[a.offsets[s.name]:a.offsets[s.name] + s.numel] = False
    for which in ("params", "slot:m", "slot:v"):
        assert not a.full(which)[pad.to(a.params.device)].any()   # nothing between or behind the tensors is touched


@pytest.mark.gpu
def test_flat_muon_matrices_by_name_and_without_any():
    named = {"g"}
    a = _arena(ODD_SPECS, "cuda")
    run_steps(a, ODD_SPECS, FlatMuon(a, matrices=named, ns_steps=3), 2, named=named, steps=3)
    a = _arena(ODD_SPECS, "cuda")
    run_steps(a, ODD_SPECS, FlatMuon(a, matrices=()), 2, named=set())
    vec = [ParamSpec("b", (70,), "ones")]
    a = _arena(vec, "cuda")
    run_steps(a, vec, FlatMuon(a), 2)


@pytest.mark.gpu
def test_flat_muon_same_state_same_bits_and_two_optimizers_at_once():
    specs = lenet_param_specs()
    arenas = [_arena(specs, "cuda") for _ in range(3)]
    opts = [FlatMuon(a) for a in arenas]
    grad = torch.randn(arenas[0].total, generator=torch.Generator().manual_seed(0)) * 1e-3
    for a in arenas:
        a.grads.copy_(grad)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in arenas]
    for _ in range(3):
        for o, s in zip(opts, streams):
            with torch.cuda.stream(s):
                o.step(0.02)
    torch.cuda.synchronize()
    for a in arenas[1:]:
        assert torch.equal(a.params, arenas[0].params) and torch.equal(a.slots["m"], arenas[0].slots["m"])


@pytest.mark.gpu
def test_flat_muon_trains_with_the_dense_layers():
    """Linear layers, their gradients and the optimizer as a program uses them: the parameters after three steps agree with the
    same program in 64 bits (bias vectors by Adam; gelu layer and a residual layer)."""
    specs = [ParamSpec("w1", (24, 72), "trunc_normal"), ParamSpec("b1", (72,), "zeros"), ParamSpec("w2", (72, 24), "trunc_normal"), ParamSpec("b2", (24,), "zeros")]
    a = _arena(specs, "cuda")
    opt = FlatMuon(a)
    p64 = {n: t.double().cpu() for n, t in a.items()}
    flat = [t.double().cpu() for t in (a.params, a.slots["m"], a.slots["v"])]
    g = torch.Generator().manual_seed(2)
    for t in range(1, 4):
        x, y = torch.randn(50, 24, generator=g), torch.randn(50, 24, generator=g)
        xg = x.cuda()
        pre = torch.empty(50, 72, device="cuda")
        h = nv.linear(xg, a.param("w1"), a.param("b1"), activation="gelu", pre=pre)
        out = nv.linear(h, a.param("w2"), a.param("b2"), residual=xg)
        dout = (out - y.cuda()) / 50
        dh, _, _ = nv.linear_bwd(dout, h, a.param("w2"), dw=a.grad("w2"), db=a.grad("b2"))
        nv.linear_bwd(dh, xg, a.param("w1"), pre=pre, activation="gelu", dx=False, dw=a.grad("w1"), db=a.grad("b1"))
        leaves = {n: v.clone().requires_grad_() for n, v in p64.items()}
        z = x.double() @ leaves["w1"] + leaves["b1"]
        o = (z * torch.special.ndtr(z)) @ leaves["w2"] + leaves["b2"] + x.double()
        (0.5 * ((o - y.double()) ** 2).sum() / 50).backward()
        grad = torch.zeros(a.total, dtype=torch.float64)
        for n, v in leaves.items():
            grad[a.offsets[n]:a.offsets[n] + v.numel()] = v.grad.reshape(-1)
            # fp32 sums of at most 72 terms on values of size one, through two layers
            assert torch.allclose(a.grad(n).double().cpu(), v.grad, rtol=1e-4, atol=2e-6)
        opt.step(0.02, vector_lr=1e-3)
        muon64(flat, specs, a.offsets, grad, t, 0.02, 1.0, 1e-3)
        p64 = {s.name: flat[0][a.offsets[s.name]:a.offsets[s.name] + s.numel].view(s.shape).clone() for s in specs}
    for n, v in p64.items():
        # gradients agree to 1e-5 of their size; small singular values may pass that on 485-fold, to lr * 5e-3
        assert torch.allclose(a.param(n).double().cpu(), v, atol=3 * 0.02 * 5e-3)


def test_flat_muon_refuses_bad_arguments():
    a = _arena(ODD_SPECS)
    with pytest.raises(ValueError):
        FlatMuon(a, matrices=["nope"])
    with pytest.raises(ValueError):
        FlatMuon(a, matrices=["b"])
    with pytest.raises(ValueError):
        FlatMuon(ParamArena(ODD_SPECS, "cpu", ("m",)))
