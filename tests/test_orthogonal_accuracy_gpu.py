"""Newton-Schulz orthogonalisation and the Muon step (csrc/orthogonal.hip): as accurate as the iteration in f32, whatever the
matrix looks like.

Tolerance.  The iteration in plain f32 (torch, on the same input) and the kernels round at the same places: X, its Gram matrix and
their products are f32 values, sums are f32.  They differ in the order of their sums and, where the kernels work on Gram matrices
alone for up to three steps, in the polynomial's form: an error of such a Gram matrix counts |b| / a times as much as one of X, twice
(from either side), below 3.  With 2 for another order of the sums and 4/3 for the largest of many errors: at most 8 times the
plain iteration's own error against 64 bits, and 4 roundings (2^-24) more where that one happens to be smaller than its rounding."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
COEFFS = (3.4445, -4.7750, 2.0315)


def iterate(g, steps=5, coeffs=COEFFS, eps=1e-7, dtype=torch.float64):
    """The plain iteration on a stack of matrices; `dtype` float64: the reference, float32: what its error is measured against."""
    x = g.to(dtype)
    tall = x.shape[-2] > x.shape[-1]
    if tall:
        x = x.mT.contiguous()
    x = x / (x.double().flatten(-2).norm(dim=-1)[..., None, None] + eps).to(dtype)
    a, b, c = coeffs
    for _ in range(steps):
        k = x @ x.mT.contiguous()
        x = a * x + (b * k + c * (k @ k)) @ x
    return x.mT.contiguous() if tall else x


def errors(got, want):
    """Relative errors of every row, of every column and of the whole: the largest of each."""
    d = got.double() - want
    return [float((d.norm(dim=k) / want.norm(dim=k)).max()) for k in (-1, -2, (-1, -2))]


def check(got, g, steps=5, coeffs=COEFFS, eps=1e-7, scale=None):
    """`scale`: a factor per entry that makes rows and columns of the result comparable (powers of two)."""
    want, plain = iterate(g, steps, coeffs, eps), iterate(g, steps, coeffs, eps, torch.float32)
    assert got.shape == g.shape and got.dtype == g.dtype
    if scale is not None:
        got, want, plain = got.double() * scale, want * scale, plain.double() * scale
    off, base = errors(got, want), errors(plain, want)
    half = 2.0 ** -8 if g.dtype == torch.bfloat16 else 0.0
    print('errors (row, column, whole):', off, 'plain f32:', base)
    for o, p in zip(off, base):
        assert o <= 8 * p + 4 * 2.0 ** -24 + half, (off, base)


def graded(count, rows, cols, kind, decades, seed=0):
    """Random matrices whose rows and / or columns span `decades` powers of ten (in powers of two), and the inverse factors."""
    gen = torch.Generator().manual_seed(seed + 7 * rows + cols)
    g = torch.randn(count, rows, cols, generator=gen)

    def factors(n, on):
        if not on:
            return torch.zeros(n)
        e = torch.linspace(0.0, -decades * math.log2(10.0), n).round() if kind.startswith('ramp') else \
            torch.where(torch.arange(n) % 2 == 0, 0.0, -round(decades * math.log2(10.0)) * 1.0)
        return e[torch.randperm(n, generator=gen)]
    e = factors(rows, 'row' in kind)[:, None] + factors(cols, 'col' in kind)[None, :]
    return (g * torch.exp2(e)).cuda(), torch.exp2(-e.double()).cuda()


# one workgroup, panels of columns, products as launches with chains of one, two and three steps; wide and tall
PATHS = [(3, 48, 100), (2, 100, 20), (2, 40, 1000), (1, 900, 30), (2, 64, 449), (2, 128, 400), (1, 300, 170), (20, 200, 1000), (8, 256, 2304), (6, 1030, 1100)]


@pytest.mark.parametrize('count,rows,cols', PATHS)
@pytest.mark.parametrize('kind', ['row', 'col', 'ramp row', 'ramp row col'])
@pytest.mark.parametrize('decades', [6, 9])
def test_graded_rows_and_columns(count, rows, cols, kind, decades):
    """Rows and columns far below the others keep their relative accuracy: the iteration commutes with neither scaling, but f32 values
    have exponents of their own."""
    from lsps_amd import ops
    g, scale = graded(count, rows, cols, kind, decades)
    check(ops.newton_schulz(g), g, scale=scale)


@pytest.mark.parametrize('count,rows,cols', [(2, 32, 64), (2, 64, 640), (1, 128, 400), (20, 200, 1000), (8, 256, 1100)])
@pytest.mark.parametrize('decades', [6, 9])
def test_graded_rows_over_many_steps(count, rows, cols, decades):
    """Twenty steps take rows of 1e-9 up to the size of the others: what they lost would be a part of the whole by then."""
    from lsps_amd import ops
    g, scale = graded(count, rows, cols, 'row', decades)
    check(ops.newton_schulz(g, 20), g, 20, scale=scale)


@pytest.mark.parametrize('count,rows,cols', [(4, 1030, 1950), (4, 1950, 1030), (1, 2250, 2250)])
def test_wide_tiles_of_odd_halves(count, rows, cols):
    """128 x 128 tiles, symmetric and not, on an odd number of 64-row and 64-column halves."""
    from lsps_amd import ops
    g = torch.randn(count, rows, cols, generator=torch.Generator().manual_seed(5)).cuda()
    check(ops.newton_schulz(g), g)


@pytest.mark.parametrize('count,rows,cols', [(2, 48, 100), (2, 40, 1000), (2, 128, 400)])
def test_graded_bf16(count, rows, cols):
    from lsps_amd import ops
    g, scale = graded(count, rows, cols, 'ramp row col', 6)
    check(ops.newton_schulz(g.bfloat16()), g.bfloat16(), scale=scale)
