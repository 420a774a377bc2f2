"""Layer norm (csrc/layernorm.hip) against its formula in 64 bits.

Tolerances.  f32 rounds by 2^-24 relative.  A normalised value is (x - mu) r: mu and the variance come from sums whose trees are
at most 16 + 6 + 4 roundings deep, so each of the few operations on the way contributes at most ~32 * 2^-24 of max|x - mu| r plus
32 * 2^-24 of max|x| r (mu's own error): F32 = 2^-19 of that size.  A bf16 result adds 2^-8 of its own value.  A sum of terms t
over a tree of depth d is off by at most d 2^-24 sum|t|."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
F32 = 2.0 ** -19
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}

# one row, one column; both sides of every width at which another variant takes over; odd, ragged and long rows
SHAPES = [(1, 1), (3, 1), (1, 2), (5, 3), (64, 50), (17, 64), (33, 65), (130, 128), (9, 129), (257, 256), (100, 257), (5, 512), (7, 513),
          (7, 1023), (13, 1024), (6, 1025), (3, 2048), (41, 2049), (19, 4096), (2, 4097), (9, 8192), (3, 8193), (2, 16384), (1, 16385),
          (5, 20001), (3, 70000), (70, 9001), (2500, 48), (20000, 7), (5000, 300), (700, 5000)]


def make(rows, cols, dtype, seed=0, offset=0.0):
    gen = torch.Generator().manual_seed(seed + rows * 131 + cols)
    x = (torch.randn(rows, cols, generator=gen) * torch.exp(0.5 * torch.randn(rows, 1, generator=gen)) + torch.randn(rows, 1, generator=gen) + offset)
    dy = torch.randn(rows, cols, generator=gen)
    w = 1.0 + 0.3 * torch.randn(cols, generator=gen)
    b = 0.3 * torch.randn(cols, generator=gen)
    return x.to(dtype).cuda(), dy.to(dtype).cuda(), w.cuda(), b.cuda()


def formula(x, w, b, eps):
    x = x.double()
    mu = x.mean(-1, keepdim=True)
    r = ((x - mu) ** 2).mean(-1, keepdim=True).add(eps).rsqrt()
    h = (x - mu) * r
    y = h * (1.0 if w is None else w.double()) + (0.0 if b is None else b.double())
    return y, h, r


def check_forward(y, x, w, b, eps=1e-5):
    want, h, r = formula(x, w, b, eps)
    wmax = 1.0 if w is None else float(w.abs().max())
    size = (h.abs().amax(-1, keepdim=True) + x.double().abs().amax(-1, keepdim=True) * r) * wmax + (0.0 if b is None else float(b.abs().max()))
    tol = F32 * size + (HALF[x.dtype] * want.abs() if x.dtype != torch.float32 else 0.0)
    assert y.shape == x.shape and y.dtype == x.dtype
    assert bool(((y.double() - want).abs() <= tol).all()), float(((y.double() - want).abs() - tol).max())


def check_backward(dx, dw, db, x, dy, w, b, eps=1e-5, depth=None):
    _, h, r = formula(x, w, b, eps)
    rows = x.shape[0]
    d = dy.double()
    g = d * (1.0 if w is None else w.double())
    m1, m2 = g.mean(-1, keepdim=True), (g * h).mean(-1, keepdim=True)
    size = h.abs().amax(-1, keepdim=True) + x.double().abs().amax(-1, keepdim=True) * r       # of a normalised value's error
    if dx is not None:
        want = r * (g - m1 - h * m2)
        gmax = g.abs().amax(-1, keepdim=True)
        # r's own relative error is F32 size^2 at most (the variance is second order in the values), h enters twice
        tol = 4 * F32 * r * gmax * (1 + size) ** 2 + (HALF[x.dtype] * want.abs() if x.dtype != torch.float32 else 0.0)
        assert dx.dtype == x.dtype and dx.shape == x.shape
        assert bool(((dx.double() - want).abs() <= tol).all()), float(((dx.double() - want).abs() - tol).max())
    depth = min(rows, 256) + 32
    if dw is not None:
        tol = depth * 2.0 ** -24 * (d * h).abs().sum(0) + F32 * (d.abs() * size).sum(0)
        assert dw.dtype == torch.float32
        assert bool(((dw.double() - (d * h).sum(0)).abs() <= tol).all())
    if db is not None:
        assert bool(((db.double() - d.sum(0)).abs() <= depth * 2.0 ** -24 * d.abs().sum(0)).all())


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('rows,cols', SHAPES)
def test_forward_and_backward(rows, cols, dtype):
    from lsps_amd import ops
    x, dy, w, b = make(rows, cols, dtype)
    for t in (x, w, b):
        t.requires_grad_(True)
    y = ops.layer_norm(x, cols, w, b)
    check_forward(y.detach(), x.detach(), w.detach(), b.detach())
    dx, dw, db = torch.autograd.grad(y, (x, w, b), dy)
    check_backward(dx, dw, db, x.detach(), dy, w.detach(), b.detach())
    again = torch.autograd.grad(ops.layer_norm(x, cols, w, b), (x, w, b), dy)
    assert all(torch.equal(p, q) for p, q in zip((dx, dw, db), again))           # no atomics


@pytest.mark.parametrize('cols', [50, 700, 3000, 18000])
@pytest.mark.parametrize('have', ['none', 'weight', 'bias'])
def test_without_parameters(cols, have):
    from lsps_amd import ops
    x, dy, w, b = make(37, cols, torch.float32)
    w, b = (w if have == 'weight' else None), (b if have == 'bias' else None)
    x.requires_grad_(True)
    leaves = [x] + [t.requires_grad_(True) for t in (w, b) if t is not None]
    y = ops.layer_norm(x, cols, w, b)
    check_forward(y.detach(), x.detach(), w, b)
    got = torch.autograd.grad(y, leaves, dy)
    check_backward(got[0], got[1] if have == 'weight' else None, got[1] if have == 'bias' else None, x.detach(), dy, w, b)


@pytest.mark.parametrize('cols', [60, 18000])
def test_only_some_gradients(cols):
    from lsps_amd import ops
    x, dy, w, b = make(70, cols, torch.float32)
    full = [t.clone().requires_grad_(True) for t in (x, w, b)]
    want = torch.autograd.grad(ops.layer_norm(full[0], cols, full[1], full[2]), full, dy)
    for k in range(3):
        t = [v.clone().requires_grad_(i == k) for i, v in enumerate((x, w, b))]
        got, = torch.autograd.grad(ops.layer_norm(t[0], cols, t[1], t[2]), t[k], dy)
        assert torch.equal(got, want[k])


def test_shapes_pitches_and_orders():
    from lsps_amd import ops
    x, dy, w, b = make(60, 84, torch.float32)
    # several normalised dimensions, several leading ones
    x4, w2 = x.view(4, 15, 12, 7), w.view(12, 7)
    y = ops.layer_norm(x4, (12, 7), w2, b.view(12, 7))
    assert y.shape == x4.shape and torch.equal(y.view(60, 84), ops.layer_norm(x, 84, w, b))
    for dtype in (torch.float32, torch.bfloat16):
        for off in (0, 1, 3):                                      # rows at a pitch, from an odd element on; every second row; a transpose
            wide = torch.full((60, 97), float('nan'), device='cuda', dtype=dtype)
            wide[:, off:off + 84] = x.to(dtype)
            for view in (wide[:, off:off + 84], wide[::2, off:off + 84], x.to(dtype).t().contiguous().t(), x.to(dtype)[:1].expand(9, 84)):
                leaf = view.detach().requires_grad_(True)
                wl = w.clone().requires_grad_(True)
                y = ops.layer_norm(leaf, 84, wl, b)
                assert y.is_contiguous()
                check_forward(y.detach(), view, w, b)
                g = torch.full((view.shape[0], 99), float('nan'), device='cuda', dtype=dtype)
                g[:, 2:86] = dy[:view.shape[0]].to(dtype)
                dx, dw = torch.autograd.grad(y, (leaf, wl), g[:, 2:86])
                check_backward(dx, dw, None, view, dy[:view.shape[0]].to(dtype), w, b)
    # a broadcast gradient (the backward of a sum)
    leaf = x.clone().requires_grad_(True)
    ops.layer_norm(leaf, 84, w, b).sum().backward()
    check_backward(leaf.grad, None, None, x, torch.ones_like(x), w, b)


def test_rows_do_not_touch_each_other_and_nothing_outside_is_written():
    """NaN and infinities stay in their rows; the bytes around views are left alone."""
    from lsps_amd import ops
    for cols in (50, 300, 5000, 17000):
        x, dy, w, b = make(23, cols, torch.float32)
        clean = ops.layer_norm(x, cols, w, b)
        bad = x.clone()
        bad[3, 7], bad[11, cols - 1], bad[22, 0] = float('nan'), float('inf'), -float('inf')
        y = ops.layer_norm(bad, cols, w, b)
        keep = [i for i in range(23) if i not in (3, 11, 22)]
        assert torch.equal(y[keep], clean[keep]) and bool(torch.isnan(y[[3, 11, 22]]).all())
        leaf = bad.requires_grad_(True)
        dx, = torch.autograd.grad(ops.layer_norm(leaf, cols, w, b), leaf, dy)
        assert bool(torch.isfinite(dx[keep]).all()) and bool(torch.isnan(dx[[3, 11, 22]]).all())


@pytest.mark.parametrize('cols', [40, 1000, 6000, 30000])
def test_constant_rows_and_large_offsets(cols):
    """A constant row has variance 0: y = b exactly, rstd = 1/sqrt(eps).  An offset 1000 times the spread costs its digits only."""
    from lsps_amd import ops
    x = torch.full((4, cols), 3.0, device='cuda')
    _, _, w, b = make(4, cols, torch.float32)
    y = ops.layer_norm(x, cols, w, b)
    # 3.0 times any column count below 2^22 sums exactly in f32, its mean is off by the one rounding of 1 / cols at most
    assert bool(((y - b).abs() <= w.abs() * (3 * 2.0 ** -23) / 1e-5 ** 0.5).all())
    x, _, w, b = make(6, cols, torch.float32, offset=1000.0)
    check_forward(ops.layer_norm(x, cols, w, b), x, w, b)


def test_gradient_against_differences():
    from lsps_amd import ops
    x, dy, w, b = make(6, 100, torch.float32)
    leaves = [t.clone().requires_grad_(True) for t in (x, w, b)]
    grads = torch.autograd.grad(ops.layer_norm(leaves[0], 100, leaves[1], leaves[2]), leaves, dy)
    gen = torch.Generator().manual_seed(5)
    step = 2.0 ** -6
    for k, base in enumerate((x, w, b)):
        v = torch.randn(base.shape, generator=gen).cuda()
        at = [t.clone() for t in (x, w, b)]
        vals = []
        for s in (step, -step):
            at[k] = base + s * v
            vals.append(float((ops.layer_norm(at[0], 100, at[1], at[2]).double() * dy.double()).sum()))
        num, ana = (vals[0] - vals[1]) / (2 * step), float((grads[k].double() * v.double()).sum())
        # rounding: every y is off by F32 * ~10 at most; truncation: step^2 / 6 of the third derivative, which is below
        # ~100 r^3 per unit of |dy| on average
        tol = float(dy.abs().sum()) * (F32 * 10 / step + step * step)
        assert abs(num - ana) <= tol and abs(ana) > tol, (k, num, ana, tol)


@pytest.mark.parametrize('rows,cols', [(9, 3), (33, 50), (7, 1023), (5, 9000), (3, 20000)])
@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
def test_without_gradients_the_same_bits(rows, cols, dtype):
    """No statistics are kept when nothing needs a gradient."""
    from lsps_amd import ops
    gen = torch.Generator().manual_seed(rows)
    x = torch.randn(rows, cols, generator=gen).to(dtype).cuda()
    w, b = torch.randn(cols, generator=gen).cuda(), torch.randn(cols, generator=gen).cuda()
    want = ops.layer_norm(x, cols, w.clone().requires_grad_(True), b)
    assert want.requires_grad and not ops.layer_norm(x, cols, w, b).requires_grad
    assert torch.equal(ops.layer_norm(x, cols, w, b), want)
    with torch.no_grad():
        assert torch.equal(ops.layer_norm(x.requires_grad_(True), cols, w, b), want)


def test_empty():
    from lsps_amd import ops
    for dtype in (torch.float32, torch.bfloat16):
        x = torch.empty(0, 5, device='cuda', dtype=dtype, requires_grad=True)
        w, b = torch.ones(5, device='cuda', requires_grad=True), torch.zeros(5, device='cuda', requires_grad=True)
        y = ops.layer_norm(x, 5, w, b)
        assert y.shape == (0, 5) and y.dtype == dtype
        y.sum().backward()
        assert x.grad.shape == (0, 5) and not w.grad.any() and not b.grad.any()


def test_other_stream_and_two_graphs():
    """On a side stream, and captured: two graphs replayed in turn with eager work between them give the eager bits each time."""
    from lsps_amd import ops
    cases = [make(300, 700, torch.float32), make(40, 20001, torch.bfloat16)]

    def step(x, dy, w, b):
        cols = w.numel()
        leaves = [t.detach().requires_grad_(True) for t in (x, w, b)]
        y = ops.layer_norm(leaves[0], cols, leaves[1], leaves[2])
        return (y.detach(),) + torch.autograd.grad(y, leaves, dy)
    want = [step(*c) for c in cases]
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = [step(*c) for c in cases]
    torch.cuda.current_stream().wait_stream(s)
    for a, b in zip(got, want):
        assert all(torch.equal(p, q) for p, q in zip(a, b))
    graphs = []
    for c in cases:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = step(*c)
        graphs.append((g, out))
    for k in range(3):
        for (g, out), c, w in zip(graphs, cases, want):
            for t in out:
                t.fill_(k)
            g.replay()
            step(*c)
            torch.cuda.synchronize()
            assert all(torch.equal(p, q) for p, q in zip(out, w))


@pytest.mark.parametrize('rows,cols', [(540001, 4096), (55000, 40001)])
def test_beyond_32_bits(rows, cols):
    """More than 2^31 elements: the first and the last rows, and the parameter gradients of a gradient that is zero but there."""
    from lsps_amd import ops
    _, _, w, b = make(1, cols, torch.float32)
    ends = torch.tensor([0, 1, rows - 2, rows - 1], device='cuda')
    x = torch.empty(rows, cols, device='cuda', dtype=torch.bfloat16).normal_()
    dy = torch.zeros_like(x)
    dy[ends] = torch.randn(4, cols, device='cuda').bfloat16()
    leaves = [x.requires_grad_(True), w.requires_grad_(True), b.requires_grad_(True)]
    y = ops.layer_norm(x, cols, w, b)
    dx, dw, db = torch.autograd.grad(y, leaves, dy)
    xe, we, be = x.detach()[ends], w.detach(), b.detach()
    check_forward(y.detach()[ends], xe, we, be)
    check_backward(dx[ends], dw, db, xe, dy[ends], we, be)
    assert not dx[2:rows - 2:997].any()


def test_differentiable_once():
    from lsps_amd import ops
    x = torch.randn(4, 10, device='cuda', requires_grad=True)
    g, = torch.autograd.grad(ops.layer_norm(x, 10).square().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()
