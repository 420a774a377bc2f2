"""Newton-Schulz orthogonalisation and the Muon step (csrc/orthogonal.hip) against the iteration in 64 bits.

Tolerance.  A matrix is held to 22 bits (2^-22 relative per rounding), a product adds that of two operands and its f32
accumulation.  An error of X or of its Gram matrix in the direction of a small singular value grows by at most `a` per step, by
at most a^steps altogether (the chain's a^4 |b| / a = 195 for three steps is below a^5 = 485): with |X0|_F <= 1 and at most 16
roundings of such weight, the result is off by no more than 16 a^steps 2^-22 in the Frobenius norm.  bf16 adds 2^-8 of the
result."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
COEFFS = (3.4445, -4.7750, 2.0315)


def iterate(g, steps=5, coeffs=COEFFS, eps=1e-7):
    x = g.double()
    tall = x.shape[-2] > x.shape[-1]
    if tall:
        x = x.mT
    x = x / (x.flatten(-2).norm(dim=-1)[..., None, None] + eps)
    a, b, c = coeffs
    for _ in range(steps):
        k = x @ x.mT.contiguous()
        x = a * x + (b * k + c * (k @ k)) @ x
    return x.mT.contiguous() if tall else x


def tolerance(want, dtype, steps=5, a=COEFFS[0]):
    return 16 * max(a, 1.0) ** steps * 2.0 ** -22 + (2.0 ** -8 * want.flatten(-2).norm(dim=-1) if dtype == torch.bfloat16 else 0.0)


def check(got, g, steps=5, coeffs=COEFFS, eps=1e-7):
    want = iterate(g, steps, coeffs, eps)
    assert got.shape == g.shape and got.dtype == g.dtype
    off = (got.double() - want).flatten(-2).norm(dim=-1)
    assert bool((off <= tolerance(want, g.dtype, steps, coeffs[0])).all()), (off, tolerance(want, g.dtype, steps, coeffs[0]))


def grads(count, rows, cols, seed=0, size=1e-3):
    gen = torch.Generator().manual_seed(seed + 7 * rows + cols)
    r = max(1, min(rows, cols) // 6)
    g = torch.randn(count, rows, r, generator=gen) @ torch.randn(count, r, cols, generator=gen) / math.sqrt(r)
    return ((g + torch.randn(count, rows, cols, generator=gen)) * size).cuda()


SHAPES = [(1, 1, 1), (2, 1, 9), (2, 9, 1), (1, 2, 3), (3, 20, 50), (1, 50, 108), (2, 64, 64), (2, 64, 49), (1, 65, 63), (1, 128, 129),
          (2, 130, 65), (5, 100, 333), (1, 333, 1021), (2, 256, 256), (1, 257, 700), (1, 20, 8192), (3, 8192, 20), (70, 33, 40), (1, 512, 513),
          (3, 64, 448), (2, 449, 64), (2, 448, 30), (300, 5, 31),
          # short sides of up to 64: panels of several widths, the last one narrow, and too many of them for panels
          (2, 64, 257), (2, 64, 449), (3, 50, 1000), (2, 9000, 33), (1, 1, 14336), (2, 3, 14337), (40, 64, 576), (150, 40, 600), (70, 64, 448),
          (300, 40, 300), (90, 20, 700),
          (40, 192, 200), (1, 1024, 1100), (20, 448, 1000),
          # 128 x 128 tiles with odd 64-row halves, symmetric and not; chains of two and three
          (40, 520, 600), (40, 200, 930), (16, 260, 1100), (6, 1030, 1100), (2, 2100, 1030), (250, 260, 450)]


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('count,rows,cols', SHAPES)
def test_newton_schulz(count, rows, cols, dtype):
    from lsps_amd import ops
    g = grads(count, rows, cols).to(dtype)
    keep = g.clone()
    out = ops.newton_schulz(g)
    check(out, g)
    assert torch.equal(g, keep) and torch.equal(out, ops.newton_schulz(g))
    assert torch.equal(ops.newton_schulz(g[0]), out[0]) or count > 1        # (another count may take another tile)


@pytest.mark.parametrize('steps', [1, 2, 3, 4, 5, 6, 7, 9])
def test_steps_and_coefficients(steps):
    from lsps_amd import ops
    g = grads(2, 70, 150)
    check(ops.newton_schulz(g, steps), g, steps)
    for coeffs in ((1.5, -0.5, 0.0), (1.875, -1.25, 0.375), (2.0, -1.5, 0.5)):
        check(ops.newton_schulz(g, steps, coeffs), g, steps, coeffs)


def test_converges_to_the_orthogonal_factor():
    """With (1.875, -1.25, 0.375), whose iterates tend to 1, enough steps give U V^T of the singular value decomposition."""
    from lsps_amd import ops
    gen = torch.Generator().manual_seed(1)
    u, _ = torch.linalg.qr(torch.randn(40, 40, generator=gen, dtype=torch.float64))
    v, _ = torch.linalg.qr(torch.randn(90, 40, generator=gen, dtype=torch.float64))
    g = (u * torch.linspace(0.5, 1.0, 40, dtype=torch.float64)) @ v.T
    out = ops.newton_schulz(g.float().cuda(), 14, (1.875, -1.25, 0.375)).cpu().double()
    # from 1 on an error is not amplified (the polynomial's slope there is 0): rounding of the last steps only
    assert float((out - u @ v.T).norm()) <= 16 * 2.0 ** -22 * 40 ** 0.5 * 4


@pytest.mark.parametrize('rows,cols', [(48, 100), (300, 170), (20, 30), (48, 700), (900, 20)])
def test_zero_tiny_huge_low_rank_and_bad_matrices(rows, cols):
    """One bad matrix of a stack leaves the others alone; sizes at the ends of f32 neither overflow nor vanish."""
    from lsps_amd import ops
    g = grads(7, rows, cols)
    clean = ops.newton_schulz(g, eps=0.0)
    g[1] = 0.0
    g[2] *= 1e-30
    g[3] *= 1e36
    g[4, 0, 0] = float('nan')
    g[5] = torch.outer(torch.randn(rows), torch.randn(cols)).cuda()
    g[6] = 0.0
    g[6, rows - 1, cols - 1] = -5.0
    out = ops.newton_schulz(g)
    assert not out[1].any() and bool(torch.isnan(out[4]).all())
    check(ops.newton_schulz(g[2:4], eps=0.0), g[2:4], eps=0.0)
    for k in (0, 5, 6):
        check(out[k], g[k])
    assert torch.equal(ops.newton_schulz(g, eps=0.0)[0], clean[0])
    g[4, 0, 0] = float('inf')
    assert bool(torch.isnan(ops.newton_schulz(g)[4]).all())


def test_views_types_and_empty():
    from lsps_amd import ops
    g = grads(6, 40, 72)
    assert torch.equal(ops.newton_schulz(g.view(2, 3, 40, 72)), ops.newton_schulz(g).view(2, 3, 40, 72))
    assert torch.equal(ops.newton_schulz(g.mT), ops.newton_schulz(g.mT.contiguous()))
    odd = torch.zeros(6 * 40 * 72 + 1, device='cuda')[1:].view(6, 40, 72)            # 4-byte aligned
    odd.copy_(g)
    assert torch.equal(ops.newton_schulz(odd), ops.newton_schulz(g))
    for shape in ((0, 3, 4), (2, 0, 4), (2, 4, 0)):
        assert ops.newton_schulz(torch.empty(shape, device='cuda')).shape == shape
    with torch.no_grad():
        p = torch.nn.Parameter(g[0].clone())
        assert torch.equal(ops.newton_schulz(p), ops.newton_schulz(g[0]))


def muon_reference(p, g, m, lr, momentum, nesterov, wd, rms, gscale, steps=5):
    p, g, m = p.double(), g.double() * gscale, m.double()
    m = momentum * m + g
    u = g + momentum * m if nesterov else m
    mat = u.reshape(u.shape[0], -1)
    o = iterate(mat, steps).reshape(u.shape)
    s = lr * rms * math.sqrt(max(mat.shape))
    return p * (1 - lr * wd) - s * o, m, s, o


SETS = [[(50, 108)], [(50, 108), (20, 50), (50, 20), (108, 50)], [(64, 1, 7, 7), (128, 64, 3, 3), (20, 48, 2, 2), (1, 9), (9, 1), (256, 300)],
        [(33 + i % 7, 20 + i) for i in range(70)],
        [(30, 40), (40, 30), (30, 40), (200, 900), (70, 30), (200, 900), (520, 2100), (400, 420), (40, 30), (192, 500)],
        [(64, 600), (20, 8192), (900, 40), (30, 40)],
        [(1100, 1030)] * 5 + [(40, 60), (1030, 1090)]]


@pytest.mark.parametrize('nesterov', [True, False])
@pytest.mark.parametrize('shapes', SETS)
def test_muon_step(shapes, nesterov):
    from lsps_amd import ops
    gen = torch.Generator().manual_seed(3)
    ps = [0.02 * torch.randn(s, generator=gen).cuda() for s in shapes]
    ms = [1e-3 * torch.randn(s, generator=gen).cuda() for s in shapes]
    gs = [1e-3 * torch.randn(s, generator=gen).cuda() for s in shapes]
    kw = dict(lr=0.03, momentum=0.9, nesterov=nesterov, weight_decay=0.1, rms=0.3, grad_scale=0.5)
    for step in range(2):
        want = [muon_reference(p, g, m, 0.03, 0.9, nesterov, 0.1, 0.3, 0.5) for p, g, m in zip(ps, gs, ms)]
        keep = [g.clone() for g in gs]
        assert ops.muon_step_(ps, gs, ms, **kw) is None
        for p, g, m, k, (wp, wm, s, o) in zip(ps, gs, ms, keep, want):
            assert torch.equal(g, k)
            assert bool(((m.double() - wm).abs() <= 2 * 2.0 ** -24 * (wm.abs() + 2e-3)).all())
            # the momentum's rounding (2^-23 relative) is one of the 16 of the iteration's bound; p itself rounds twice
            off = float((p.double() - wp).norm())
            assert off <= s * tolerance(o.reshape(o.shape[0], -1), torch.float32) + 2.0 ** -23 * float(wp.norm()), (tuple(p.shape), off)


def test_muon_step_equals_its_parts():
    """One call over many matrices, calls one by one and newton_schulz give the same update."""
    from lsps_amd import ops
    g = [grads(1, r, c, seed=r)[0] for r, c in ((40, 90), (200, 60), (64, 64))]
    p0 = [torch.zeros_like(t) for t in g]
    m0 = [torch.zeros_like(t) for t in g]
    ops.muon_step_(p0, g, m0, lr=1.0, momentum=0.0, nesterov=False, rms=1.0)
    for p, t, m in zip(p0, g, m0):
        assert torch.equal(m, t)
        s = math.sqrt(max(t.shape))
        want = -s * ops.newton_schulz(t).double()
        assert float((p.double() - want).norm()) <= 2 * s * tolerance(want, torch.float32) + 2.0 ** -23 * float(want.norm())


def test_streams_and_graphs():
    from lsps_amd import ops
    shapes = [(64, 49), (130, 200), (20, 300)]
    gs = [grads(1, *s)[0] for s in shapes]

    def fresh():
        return [torch.full(s, 0.5, device='cuda') for s in shapes], [torch.zeros(s, device='cuda') for s in shapes]

    def run(n):
        p, m = fresh()
        for _ in range(n):
            ops.muon_step_(p, gs, m, lr=0.1)
        return p + m
    want = [run(n) for n in (1, 2, 3)]
    wide = grads(3, 40, 1000)
    ns, nw = ops.newton_schulz(gs[1]), ops.newton_schulz(wide)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        side = run(3)
    torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(a, b) for a, b in zip(side, want[2]))
    p, m = fresh()
    g1, g2 = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(g1):
        ops.muon_step_(p, gs, m, lr=0.1)
    with torch.cuda.graph(g2):
        out = ops.newton_schulz(gs[1])
        out_wide = ops.newton_schulz(wide)
    for k in range(3):
        out.zero_()
        out_wide.zero_()
        g1.replay()
        g2.replay()
        run(1)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(p + m, want[k])) and torch.equal(out, ns) and torch.equal(out_wide, nw)


def test_two_threads_at_once():
    """Two host threads, each with a stream and matrices of its own: the same bits as one after the other."""
    import threading

    from lsps_amd import ops
    work = [[grads(1, *s, seed=k)[0] for s in ((60, 90), (130, 200), (40, 1000))[k:] + ((300, 320),)] for k in range(2)]

    def run(gs):
        p, m = [torch.full_like(g, 0.5) for g in gs], [torch.zeros_like(g) for g in gs]
        for _ in range(8):
            ops.muon_step_(p, gs, m, lr=0.1)
            x = ops.layer_norm(p[0], p[0].shape[-1])
        return p + m + [x, ops.newton_schulz(gs[-1])]
    want = [run(gs) for gs in work]
    torch.cuda.synchronize()
    got = [None, None]

    def thread(k):
        s = torch.cuda.Stream()
        with torch.cuda.stream(s):
            got[k] = run(work[k])
        s.synchronize()
    threads = [threading.Thread(target=thread, args=(k,)) for k in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join(60)
    assert all(g is not None and all(torch.equal(a, b) for a, b in zip(g, w)) for g, w in zip(got, want))



def test_beyond_32_bits():
    """A stack whose working matrices pass 4 GiB: the last matrix is the one computed alone."""
    from lsps_amd import ops
    g = torch.randn(300, 1024, 1000, device='cuda')
    out = ops.newton_schulz(g)
    for k in (0, 299):
        check(out[k], g[k])


def test_version_counters_move():
    from lsps_amd import ops
    g = grads(1, 8, 9)[0]
    p, m = torch.nn.Parameter(torch.zeros(8, 9, device='cuda')), torch.zeros(8, 9, device='cuda')
    v = p._version
    ops.muon_step_([p], [g], [m], lr=0.1)
    assert p._version > v


# ---- FlatMuon and the trainer -----------------------------------------------------------------------------------------------
def test_flat_muon_matches_its_parts():
    """Matrices step by Muon, vectors by Adam (as FlatAdam steps them), untouched parameters not at all; state dicts round-trip."""
    from lsps_amd import optim
    gen = torch.Generator().manual_seed(9)
    shapes = [(30, 8, 3, 3), (30,), (12, 50), (1, 40), (12,)]
    init = [0.1 * torch.randn(s, generator=gen) for s in shapes]

    def build(cls, **kw):
        ps = [torch.nn.Parameter(t.clone().cuda()) for t in init]
        opt = cls(ps, lr=0.01, betas=(0.5, 0.999), weight_decay=0.01, **kw)
        opt.attach()
        return ps, opt
    pm, om = build(optim.FlatMuon, momentum=0.9, rms=0.3)
    pa, oa = build(optim.FlatAdam)
    wp, wm = init[0].cuda(), torch.zeros(shapes[0], device='cuda')
    for step in range(3):
        g = [1e-2 * torch.randn(s, generator=gen).cuda() for s in shapes]
        for ps, opt in ((pm, om), (pa, oa)):
            opt.zero_grad()
            sum((p * t).sum() for i, (p, t) in enumerate(zip(ps, g)) if i != 2).backward()      # parameter 2 takes no part
            opt.step()
        wp, wm, s, o = muon_reference(wp, g[0], wm, 0.01, 0.9, True, 0.01, 0.3, 1.0)
        assert float((pm[0].detach().double() - wp).norm()) <= (step + 1) * (s * tolerance(o.reshape(30, -1), torch.float32) + 2.0 ** -23 * float(wp.norm()))
        assert torch.equal(pm[2].detach().cpu(), init[2])
        for i in (1, 3, 4):
            assert torch.equal(pm[i], pa[i])
    sd = om.state_dict()
    assert set(sd['state'][0]) == {'step', 'momentum_buffer'} and sd['state'][0]['step'] == 3 and sd['state'][2]['step'] == 0
    assert set(sd['state'][1]) == {'step', 'exp_avg', 'exp_avg_sq'}
    sd = {'state': {k: {n: (v.clone() if torch.is_tensor(v) else v) for n, v in st.items()} for k, st in sd['state'].items()},
          'param_groups': sd['param_groups']}
    for before in (True, False):                                  # loaded before and after the arena exists
        ps = [torch.nn.Parameter(p.detach().clone()) for p in pm]
        opt = optim.FlatMuon(ps, lr=0.01, betas=(0.5, 0.999), weight_decay=0.01)
        if before:
            opt.load_state_dict(sd)
        opt.attach()
        if not before:
            opt.load_state_dict(sd)
        assert opt.param_groups[0]['momentum'] == 0.9 and torch.equal(opt.flat_m, om.flat_m) and torch.equal(opt.flat_v, om.flat_v)
        assert opt.state[ps[0]]['momentum_buffer'].data_ptr() == opt.flat_m.data_ptr()
    # an Adam state: the vectors' moments, no momentum
    ps = [torch.nn.Parameter(p.detach().clone()) for p in pm]
    opt = optim.FlatMuon(ps, lr=0.01)
    opt.attach()
    opt.load_state_dict(oa.state_dict())
    assert not opt.state[ps[0]]['momentum_buffer'].any() and torch.equal(opt.state[ps[1]]['exp_avg'], oa.state[pa[1]]['exp_avg'])


@pytest.mark.parametrize('before', [True, False])
def test_adam_starts_over_with_matrices_of_a_muon_state(before):
    """A FlatMuon's matrices have no moments: their first Adam step is one of a new optimizer, vectors go on where they were."""
    from lsps_amd import optim
    gen = torch.Generator().manual_seed(4)
    shapes = [(12, 20), (12,)]
    init = [0.1 * torch.randn(s, generator=gen) for s in shapes]
    grad = [1e-2 * torch.randn(s, generator=gen).cuda() for s in shapes]

    def build(cls, sd=None, loaded_first=False):
        ps = [torch.nn.Parameter(t.clone().cuda()) for t in init]
        opt = cls(ps, lr=0.01)
        if sd and loaded_first:
            opt.load_state_dict(sd)
        opt.attach()
        if sd and not loaded_first:
            step(ps, opt)                                          # (moments that the load has to replace)
            with torch.no_grad():
                for p, t in zip(ps, init):
                    p.copy_(t.cuda())
            opt.load_state_dict(sd)
        return ps, opt

    def step(ps, opt):
        opt.zero_grad()
        sum((p * g).sum() for p, g in zip(ps, grad)).backward()
        opt.step()
    pm, om = build(optim.FlatMuon)
    for _ in range(5):
        step(pm, om)
    ps, opt = build(optim.FlatAdam, om.state_dict(), before)
    assert set(opt.state[ps[0]]) == {'step', 'exp_avg', 'exp_avg_sq'} and opt.state[ps[0]]['step'] == 0 and opt.state[ps[1]]['step'] == 5
    assert torch.equal(opt.state[ps[1]]['exp_avg'], om.state[pm[1]]['exp_avg'])
    pn, new = build(optim.FlatAdam)
    step(ps, opt)
    step(pn, new)
    assert torch.equal(ps[0], pn[0]) and not torch.equal(ps[1], pn[1])


def test_training_steps_with_layer_norm_and_muon():
    """The pose VAE with layer-normed hidden layers, stepped by FlatMuon through the trainer: the gradients and the first step are
    those of the plain computation in 64 bits; pretraining steps of the nets run on the same optimizer."""
    import cases
    import lsps_amd.trainers as prod
    from oracle import lsps_ref
    hp = dict(cases.hp_for('tiny'))
    hp['vae'] = dict(hp['vae'], norm='layer')
    hp['optimizer'] = 'muon'
    torch.manual_seed(0)
    tr = prod.LSPSTrainer(hp)
    tr.cuda(0)
    vae = tr.vae
    y = torch.randn(16, hp['vae']['input_dim'], device='cuda')
    noise = 0.05 * torch.randn(16, hp['vae']['z_dim'], device='cuda')
    tr.vae_opt.zero_grad()
    rec, z, mu, sd = vae(y, noise)
    loss = (rec - y).square().mean() + 0.1 * (mu.square().mean() + sd.square().mean())
    loss.backward()
    P = dict((n, p.detach().double().clone().requires_grad_(True)) for n, p in vae.named_parameters())

    def hidden(x, name):
        h = x @ P[name + '.model.0.weight'].T.contiguous() + P[name + '.model.0.bias']
        h = (h - h.mean(1, keepdim=True)) / torch.sqrt(h.var(1, unbiased=False, keepdim=True) + 1e-5)
        return torch.nn.functional.leaky_relu(h * P[name + '.model.1.weight'] + P[name + '.model.1.bias'], 0.01)
    h = hidden(y.double(), 'en_fc1')
    mu64 = h @ P['en_mu.weight'].T.contiguous() + P['en_mu.bias']
    sd64 = torch.nn.functional.softplus(h @ P['en_sigma.weight'].T.contiguous() + P['en_sigma.bias'])
    rec64 = hidden(mu64 + sd64 * noise.double(), 'de_fc1') @ P['de_fc2.weight'].T.contiguous() + P['de_fc2.bias']
    loss64 = (rec64 - y.double()).square().mean() + 0.1 * (mu64.square().mean() + sd64.square().mean())
    want = torch.autograd.grad(loss64, list(P.values()))
    # f32 sums over at most 108 x 16 terms through four layers: 2^-24 * 1024 of the largest gradient of a tensor
    for (n, p), w in zip(vae.named_parameters(), want):
        assert float((p.grad.double() - w).abs().max()) <= 2.0 ** -14 * float(w.abs().max()), n
    before = dict((n, p.detach().clone()) for n, p in vae.named_parameters())
    grad = dict((n, p.grad.clone()) for n, p in vae.named_parameters())
    tr.vae_opt.step()
    g = tr.vae_opt.param_groups[0]
    assert type(tr.vae_opt).__name__ == 'FlatMuon'
    for n, p in vae.named_parameters():
        if p.dim() == 2:
            wp, _, s, o = muon_reference(before[n], grad[n], torch.zeros_like(p), g['lr'], 0.95, True, g['weight_decay'], 0.2, 1.0)
            assert float((p.detach().double() - wp).norm()) <= s * tolerance(o, torch.float32) + 2.0 ** -23 * float(wp.norm()), n
        else:
            assert float((p.detach() - before[n]).abs().max()) > 0, n
    b = cases.make_inputs(2)
    A = cases.NativeAdapter(prod, 'cuda')
    tr2 = A.make_trainer(dict(cases.hp_for('tiny'), optimizer='muon'), cases.make_weights(cases.hp_for('tiny'), lsps_ref))
    old = tr2.dis_opt.arena.flat_p.clone(), tr2.gen_opt.arena.flat_p.clone()
    A.dis_update(tr2, b, hp, cases.noise(cases.latent_shape(hp, 4), 11))
    A.gen_update(tr2, b, hp, (cases.noise(cases.latent_shape(hp, 4), 12), cases.noise(cases.latent_shape(hp, 2), 13), cases.noise(cases.latent_shape(hp, 2), 14)))
    for o, opt in zip(old, (tr2.dis_opt, tr2.gen_opt)):
        assert bool(torch.isfinite(opt.arena.flat_p).all()) and not torch.equal(o, opt.arena.flat_p)
