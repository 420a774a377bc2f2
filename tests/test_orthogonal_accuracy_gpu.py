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


@pytest.mark.parametrize('rows,cols', [(21000, 22000), (22000, 20500)])
def test_matrix_whose_limbs_pass_2_gib(rows, cols):
    """One step of a matrix of 2.7 GB of limbs, against the formula applied to a vector: a missing chunk of 32 columns would be off
    by 1e-3 of it; a sum of up to 22000 terms takes 1400 roundings in runs of 16, whose errors of 2^-24 add up to about their root's
    number: 40 * 2^-24 < 2^-18."""
    from lsps_amd import ops
    gen = torch.Generator(device='cuda').manual_seed(2)
    g = torch.randn(rows, cols, generator=gen, device='cuda')
    out = ops.newton_schulz(g, 1)

    def times(m, v, transposed=False):                       # in 64 bits, a block of rows at a time
        parts = [(p.double().T.contiguous() @ v[k * 2048:k * 2048 + len(p)]) if transposed else p.double() @ v
                 for k, p in enumerate(m.split(2048))]
        return sum(parts) if transposed else torch.cat(parts)
    norm = math.sqrt(sum(float(p.double().square().sum()) for p in g.split(2048))) + 1e-7
    tall = rows > cols
    v = torch.randn(rows if tall else cols, generator=gen, device='cuda', dtype=torch.float64)
    a, b, c = COEFFS
    y = times(g, v, tall) / norm                              # X v, X with its short side in rows
    up = lambda u: times(g, times(g, u, not tall), tall) / norm ** 2           # noqa: E731     A u
    ay = up(y)
    want = a * y + b * ay + c * up(ay)
    assert float((times(out, v, tall) - want).norm()) <= 2.0 ** -18 * float(want.norm())


def gradients(count, rows, cols, seed=0):
    """Low rank under noise, as weights' gradients are."""
    gen = torch.Generator().manual_seed(seed + 7 * rows + cols)
    r = max(1, min(rows, cols) // 6)
    g = torch.randn(count, rows, r, generator=gen) @ torch.randn(count, r, cols, generator=gen) / math.sqrt(r)
    return ((g + torch.randn(count, rows, cols, generator=gen)) * 1e-3).cuda()


@pytest.mark.parametrize('count,rows,cols', [
    # one workgroup: short sides on both sides of 32, up to 320 columns; panels of several widths; products: few tiles and many, split
    # reductions, chains of one, two and three steps, 64- and 128-wide tiles
    (3, 20, 50), (1, 50, 108), (2, 31, 33), (2, 64, 64), (2, 33, 319), (2, 320, 64), (300, 40, 300), (2, 64, 321), (1, 20, 8192), (3, 50, 1000),
    (2, 9000, 33), (1, 32, 700), (3, 31, 704), (2, 705, 32), (2, 700, 20), (300, 30, 400), (5, 7, 321), (40, 64, 576), (25, 64, 640), (70, 64, 448), (1, 65, 63), (1, 65, 700), (2, 130, 65), (4, 128, 576), (5, 100, 333), (1, 333, 1021),
    (1, 200, 4000), (2, 256, 256), (1, 257, 700), (20, 448, 1000), (20, 200, 1000), (8, 256, 2304), (40, 520, 600), (1, 1024, 1100), (4, 1030, 1030)])
def test_as_accurate_as_f32(count, rows, cols):
    from lsps_amd import ops
    g = gradients(count, rows, cols)
    check(ops.newton_schulz(g), g)


EPS_PATHS = [(2, 48, 100), (2, 100, 20), (2, 40, 1000), (1, 900, 30), (2, 128, 400), (1, 300, 170)]


@pytest.mark.parametrize('count,rows,cols', EPS_PATHS)
@pytest.mark.parametrize('size', [0.1, 1.0, 10.0])
@pytest.mark.parametrize('eps', [1e-7, 0.5])
def test_eps_beside_the_norm(count, rows, cols, size, eps):
    """|G|_F of a tenth of eps to ten times it: eps counts once per matrix, whatever path computes it."""
    from lsps_amd import ops
    g = gradients(count, rows, cols)
    g *= size * eps / g.flatten(1).norm(dim=1)[:, None, None]
    check(ops.newton_schulz(g, eps=eps), g, eps=eps)
    p, m = [torch.zeros_like(t) for t in g], [torch.zeros_like(t) for t in g]
    ops.muon_step_(p, list(g), m, lr=1.0, momentum=0.0, nesterov=False, rms=1.0, eps=eps)
    check(torch.stack(p) / -math.sqrt(max(rows, cols)), g, eps=eps)


# more matrices than travel in a launch's arguments (16), than one launch enters into the table (96), than a pass takes (1024), more
# shapes than a pass takes (16)
MANY = {'40 small': [(40, 24, 50)], '40 panels': [(40, 30, 700)], '40 products': [(40, 70, 90)], '130 small of two shapes': [(65, 24, 50), (65, 40, 20)],
        '120 panels and small': [(100, 20, 330), (20, 330, 20)], '1100 tiny': [(600, 20, 24), (500, 30, 20)],
        '1060 products': [(1060, 66, 70)], '19 shapes': [(2, 66 + k, 300 - 9 * k) for k in range(19)],
        'long reductions in company': [(2, 300, 4100), (1, 20, 8192), (6, 256, 700), (1, 4500, 130)],
        '18 shapes of panels': [(1, 20 + k, 340 + 9 * k) for k in range(18)]}


@pytest.mark.parametrize('name', list(MANY))
def test_many_matrices(name):
    from lsps_amd import ops
    stacks = [gradients(*s, seed=k) for k, s in enumerate(MANY[name])]
    where = [(k, i) for k, s in enumerate(stacks) for i in range(len(s))]
    order = torch.randperm(len(where), generator=torch.Generator().manual_seed(1)).tolist()
    where = [where[i] for i in order]                         # shapes in no order
    ps = [torch.zeros_like(s) for s in stacks]
    ms = [torch.full_like(s, 1e-3) for s in stacks]
    ops.muon_step_([ps[k][i] for k, i in where], [stacks[k][i] for k, i in where], [ms[k][i] for k, i in where], lr=1.0, momentum=0.5, rms=1.0)
    for p, g, m in zip(ps, stacks, ms):
        new = 0.5 * torch.full_like(g, 1e-3).double() + g.double()
        # a product and a sum: 2^-24 of the momentum and of what is added to it
        assert bool(((m.double() - new).abs() <= 2.0 ** -23 * (new.abs() + 1e-3)).all())
        u = (g + 0.5 * m)
        check(p / -math.sqrt(max(g.shape[1:])), u)
