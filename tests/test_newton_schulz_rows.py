"""Newton-Schulz row by row and column by column: rows far below the others are results too.

With X = G / |G| and s the largest singular value that occurs (top of the sequence), row i goes x_i <- x_i p(X^T X), p(t) = a + b t + c t^2: by a
factor of F = max |p| at most, and a small row stays in proportion. fp32 products keep its relative error. Pairs h + l of fp16 (the default) keep
22 bits of an element down to a floor: half a step of fp16's smallest numbers, 2^-25, over the power of two that a matrix is kept by, so
2^-38 for X (kept times 2^13) and 2^-37 for A and P (times 2^12). An element of X adds its floor itself, an element of A or P what it does to the
row: in the 2-norm, per step,
    f = 2^-38 sqrt(c) + 2^-37 sqrt(r) s (1 + |b| + |c| s^2),      floor <- F floor + f,
from the split of X_0 (2^-38 sqrt(c)) on. Columns gather the same floors over r elements instead of c. On top of that the relative part: 2^-20 (the pairs'
few 2^-22 a step), and four times the error that the plain formula in fp32 leaves in the same row (sums in another order leave errors of that size)."""
import math

import pytest
import torch

from distributed_tensorflow_amd.models.lenet import lenet_param_specs
from distributed_tensorflow_amd.models.resnet import resnet_param_specs
from distributed_tensorflow_amd.ops import native as nv
from distributed_tensorflow_amd.ops import reference as ref
from distributed_tensorflow_amd.optim import FlatMuon
from distributed_tensorflow_amd.runtime.arena import ParamSpec
from test_newton_schulz import DTYPES, ODD_SPECS, SHAPES as NS_SHAPES, _arena, check, gradient, run_steps


def plain(g, dtype, steps=5, coeffs=ref.NS_COEFFS):
    x = g.to(dtype)
    flip = x.shape[0] > x.shape[1]
    x = x.t() if flip else x
    x = x / (x.double().norm() + 1e-7).to(dtype)
    a, b, c = coeffs
    for _ in range(steps):
        m = x @ x.t()
        x = a * x + (b * m + c * m @ m) @ x
    return (x.t() if flip else x).double()


def floors(r, c, steps=5, coeffs=ref.NS_COEFFS):
    """(floor of a row of the r x c orientation, of a column)"""
    a, b, cc = coeffs
    row, col, top = 2.0 ** -38 * math.sqrt(c), 2.0 ** -38 * math.sqrt(r), 1.001
    for _ in range(steps):
        s = torch.linspace(0, top, 2001, dtype=torch.float64)
        grow = float((a + b * s ** 2 + cc * s ** 4).abs().max())
        mix = 2.0 ** -37 * math.sqrt(r) * top * (1 + abs(b) + abs(cc) * top ** 2)
        row, col = grow * row + 2.0 ** -38 * math.sqrt(c) + mix, grow * col + 2.0 ** -38 * math.sqrt(r) + mix
        top = 1.001 * float((s * (a + b * s ** 2 + cc * s ** 4)).abs().max())
    return row, col


def matrix(m, n, scale, which, seed=0):
    """Rows 1 and 5 (or columns) times scale, row 3 exactly zero."""
    g = torch.randn(m, n, generator=torch.Generator().manual_seed(seed))
    v = g if which == "row" else g.t()
    v[1] *= scale
    v[5] *= scale
    v[3] = 0
    return g


def check_lines(out, g, which, floor):
    want, rough = plain(g, torch.float64), plain(g, torch.float32)
    lines = (lambda t: t) if which == "row" else (lambda t: t.t())
    off, fp32, size = (lines(t).norm(dim=1) for t in (out.double().cpu() - want, rough - want, want))
    limit = 4 * fp32 + 2.0 ** -20 * size + floor
    assert not lines(out)[3].any()
    worst = int((off - limit).argmax())
    assert bool((off <= limit).all()), f"{which} {worst}: off by {float(off[worst])}, at most {float(limit[worst])} (size {float(size[worst])})"


SHAPES = [(16, 300), (30, 30), (64, 256), (256, 64), (130, 300), (520, 264), (128, 1600)]   # one workgroup and tiles, X X^T whole and in parts


@pytest.mark.gpu
@pytest.mark.parametrize("which", ["row", "column"])
@pytest.mark.parametrize("scale", [1e-2, 1e-4, 1e-6, 1e-8])
@pytest.mark.parametrize("m,n", SHAPES)
def test_pairs_keep_rows_down_to_their_floor(m, n, scale, which):
    g = matrix(m, n, scale, which, seed=m + n)
    row, col = floors(min(m, n), max(m, n))
    check_lines(nv.newton_schulz(g.cuda()), g, which, row if (which == "row") == (m <= n) else col)


@pytest.mark.gpu
@pytest.mark.parametrize("which", ["row", "column"])
@pytest.mark.parametrize("scale", [1e-2, 1e-4, 1e-8, 1e-15])
@pytest.mark.parametrize("m,n", SHAPES + [(1000, 1100)])
def test_fp32_products_keep_rows_of_any_size(m, n, scale, which):
    g = matrix(m, n, scale, which, seed=m + n)
    check_lines(nv.newton_schulz(g.cuda(), products="fp32"), g, which, 0.0)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m,n", NS_SHAPES)
def test_fp32_products_shapes(m, n, dtype):
    g = gradient(m, n, seed=m * 7 + n, scale=1.0 if dtype == torch.float16 else 1e-3).to(dtype).cuda()
    keep = g.clone()
    out = nv.newton_schulz(g, products="fp32")
    assert out.dtype == dtype and torch.equal(g, keep)
    check(out, g)
    assert torch.equal(out, nv.newton_schulz(g, products="fp32"))


@pytest.mark.gpu
@pytest.mark.parametrize("m,n", [(1500, 2600), (2600, 1111), (3000, 3000), (70, 9000), (3, 40000)])
def test_fp32_products_large(m, n):
    g = gradient(m, n, seed=3, scale=1.0).cuda()
    check(nv.newton_schulz(g, products="fp32"), g)


@pytest.mark.gpu
@pytest.mark.parametrize("scale", [1e18, 1e-6, 1e-9, 1e-20, 1e-38])
def test_fp32_products_norms_far_from_one(scale):
    for m, n in ((40, 72), (130, 200)):
        g = (gradient(m, n, seed=4, scale=1.0) * scale).cuda()
        check(nv.newton_schulz(g, products="fp32"), g)


@pytest.mark.gpu
@pytest.mark.parametrize("products", nv.PRODUCTS)
@pytest.mark.parametrize("batch,m,n", [(3, 128, 1600), (2, 1000, 300), (5, 70, 90), (2, 65, 800), (6, 576, 64), (40, 20, 200)])
def test_batches_beyond_one_workgroup(batch, m, n, products):
    """Batched tiles, and X X^T of a batch in parts (the first two): every matrix of the batch by itself against 64 bits, and in its own memory."""
    g = gradient(m, n, seed=batch, batch=batch).cuda()
    g[1] *= 1e4
    store = torch.full((batch, m + 1, n + 3), 7.0, device="cuda")
    ws = torch.empty(nv.newton_schulz_workspace(m, n, batch, products) + 64, device="cuda", dtype=torch.uint8)
    ws[-64:] = 99
    out = nv.newton_schulz(g, out=store[:, :m, :n], products=products, workspace=ws[:-64])
    for i in range(batch):
        check(out[i], g[i])
    assert bool((store[:, m] == 7).all()) and bool((store[:, :, n:] == 7).all()) and bool((ws[-64:] == 99).all())
    assert torch.equal(out, nv.newton_schulz(g, products=products))   # fixed orders


@pytest.mark.gpu
def test_batches_of_the_one_workgroup_kernel_do_not_change_a_matrix():
    for m, n in ((576, 64), (48, 40), (20, 200)):
        for batch in (2, 6, 40):
            g = gradient(m, n, seed=batch, batch=batch).cuda()
            out = nv.newton_schulz(g)
            for i in range(batch):
                assert torch.equal(out[i], nv.newton_schulz(g[i]))


@pytest.mark.gpu
def test_fp32_products_special_matrices_and_replay():
    for m, n in ((40, 30), (200, 130)):
        assert not nv.newton_schulz(torch.zeros(m, n, device="cuda"), products="fp32").any()
        b = gradient(m, n, batch=3).cuda()
        clean = nv.newton_schulz(b, products="fp32")
        b[1, 5, 6] = float("nan")
        out = nv.newton_schulz(b, products="fp32")
        assert bool(out[1].isnan().all()) and torch.equal(out[0], clean[0]) and torch.equal(out[2], clean[2])
        g = gradient(m, n).cuda()
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            nv.newton_schulz(g, products="fp32")
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=s):
                held = nv.newton_schulz(g, products="fp32")
        torch.cuda.current_stream().wait_stream(s)
        for seed in range(3):
            g.copy_(gradient(m, n, seed=30 + seed).cuda())
            want = nv.newton_schulz(g, products="fp32")
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(held, want)


@pytest.mark.gpu
@pytest.mark.parametrize("specs", [ODD_SPECS, lenet_param_specs(), resnet_param_specs(1)])
def test_flat_muon_with_fp32_products(specs):
    a = _arena(specs, "cuda")
    run_steps(a, specs, FlatMuon(a, ns_products="fp32"), 2)
    pad = torch.ones(a.capacity, dtype=torch.bool)
    for s in specs:
        pad[a.offsets[s.name]:a.offsets[s.name] + s.numel] = False
    for which in ("params", "slot:m", "slot:v"):
        assert not a.full(which)[pad.to(a.params.device)].any()


@pytest.mark.gpu
@pytest.mark.parametrize("m,n", [(64, 256), (300, 140)])
def test_flat_muon_with_fp32_products_keeps_small_rows(m, n):
    """The update of a parameter that starts at zero is the result of newton_schulz, line by line (rounded by the update once more)."""
    specs = [ParamSpec("w", (m, n), "zeros")]
    a = _arena(specs, "cuda")
    g = matrix(m, n, 1e-8, "row", seed=1)
    a.grad("w").copy_(g)
    FlatMuon(a, nesterov=False, ns_products="fp32").step(1.0)
    check_lines(-a.param("w") / math.sqrt(max(1.0, n / m)), g, "row", 0.0)


def test_unknown_products_are_refused():
    for call in (lambda: nv.newton_schulz(torch.zeros(4, 4), products="fp16"), lambda: nv.newton_schulz_workspace(4, 4, products="tf32"),
                 lambda: FlatMuon(_arena([ParamSpec("w", (4, 4), "ones")]), ns_products="bf16")):
        with pytest.raises(ValueError, match="products"):
            call()


def test_fp32_products_workspace():
    """The same place as pairs take, but for matrices that pairs do in one workgroup and fp32 numbers in parts."""
    if nv._hip is None:
        pytest.skip("extension not built")
    assert nv.newton_schulz_workspace(1000, 1000, products="fp32") >= nv.newton_schulz_workspace(1000, 1000) > 2 * 4 * 1000 * 1000
    assert nv.newton_schulz_workspace(64, 768, products="fp32") >= nv.newton_schulz_workspace(64, 768)
