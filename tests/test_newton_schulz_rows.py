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

from distributed_tensorflow_amd.ops import native as nv
from distributed_tensorflow_amd.ops import reference as ref


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
