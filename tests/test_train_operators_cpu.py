"""Layer norm, Newton-Schulz and Muon without a GPU: what the entry points refuse, how FlatMuon sorts parameters, the algebra the
kernels rest on (Gram-matrix chains, two f16 limbs) in numpy."""
import ctypes

import numpy as np
import pytest
import torch

from lsps_amd import _lib, ops, optim


def err():
    return _lib.lib().lsps_last_error().decode()


def test_refusals_of_the_python_entry_points():
    x = torch.randn(3, 4)
    for bad in (lambda: ops.layer_norm(x, 5), lambda: ops.layer_norm(x, ()), lambda: ops.layer_norm(x, (2, 3, 4)),
                lambda: ops.layer_norm(x.double(), 4), lambda: ops.layer_norm(x.half(), 4), lambda: ops.layer_norm(torch.empty(3, 0), 0),
                lambda: ops.layer_norm(x, 4, torch.ones(3)), lambda: ops.layer_norm(x, 4, torch.ones(4).bfloat16()),
                lambda: ops.layer_norm(x, 4, None, torch.ones(4, 1)), lambda: ops.layer_norm(x, 4),            # no CPU fallback
                lambda: ops.newton_schulz(x[0]), lambda: ops.newton_schulz(x.double()), lambda: ops.newton_schulz(x),
                lambda: ops.newton_schulz(x.clone().requires_grad_(True)),
                lambda: ops.muon_step_([x], [x, x], [x], lr=0.1), lambda: ops.muon_step_([x], [x[0]], [x], lr=0.1),
                lambda: ops.muon_step_([x[0]], [x[0]], [x[0]], lr=0.1), lambda: ops.muon_step_([x], [x.clone()], [x.clone()], lr=0.1)):
        with pytest.raises(_lib.LspsHipError):
            bad()
    assert ops.muon_step_([], [], [], lr=0.1) is None
    assert ops._ints('t', 5, (1 << 31) - 1, -3) == (5, (1 << 31) - 1, -3)
    for n in (1 << 31, (1 << 32) + 5, -(1 << 31) - 1):                        # a C int would be another size
        with pytest.raises(_lib.LspsHipError):
            ops._ints('t', 2, n)


@pytest.mark.parametrize('more', [0, 40])
def test_overlapping_matrices_are_refused(more):
    """What a Muon step writes (weights, momenta) may not overlap anything else of it; gradients may be shared.  The addresses are
    never followed: a call that passes ends at the missing workspace."""
    h = _lib.lib()
    far = [(1 << 30) + k * 4096 for k in range(3 * more)]                   # (more matrices than the check keeps on its stack)

    def step(*mats):
        mats = [_lib.LspsMuonMatrix(*m) for m in mats] + [_lib.LspsMuonMatrix(*far[3 * k:3 * k + 3], 4, 8) for k in range(more)]
        return h.lsps_muon_step((_lib.LspsMuonMatrix * len(mats))(*mats), len(mats), 0.1, 0.9, 1, 0.0, 0.2, 1.0, 5, 3.4445, -4.775, 2.0315, 1e-7,
                                None, 0, None)
    a, size = 4096, 4 * 4 * 8
    assert step((a, a + size, a + 2 * size, 4, 8)) == -2
    assert step((a, a + size, a + 2 * size, 4, 8), (a + 4 * size, a + 3 * size, a + 6 * size, 4, 8)) == -2
    assert step((a, a + size, a + 2 * size, 4, 8), (a + 4 * size, a + size, a + 5 * size, 4, 8)) == -2      # one gradient for two weights
    for p, g, m in ((a, a, a + size), (a, a + size, a), (a, a + size, a + 4), (a, a + size - 4, a + 4 * size), (a + size - 4, a, a + 4 * size)):
        assert step((p, g, m, 4, 8)) == -1 and 'overlap' in err(), (p, g, m)
    assert step((a, a + size, a + 2 * size, 4, 8), (a + 4 * size, a + 5 * size, a, 4, 8)) == -1             # one weight is another's momentum
    assert step((a, a + 9 * size, a + 3 * size, 4, 8), (a + size // 2, a + 5 * size, a + 6 * size, 2, 2)) == -1


def test_refusals_of_the_c_entry_points():
    """Arguments are checked before anything touches the device (there is none here)."""
    h = _lib.lib()
    buf = (ctypes.c_char * 256)()
    p = ctypes.cast(buf, ctypes.c_void_p)

    def ln(rows=2, cols=8, ldx=8, dtype=0, eps=1e-5, x=p, y=p, mean=p, ws=None, n=0):
        return h.lsps_layernorm_fwd(x, None, None, y, mean, p, rows, cols, ldx, dtype, eps, ws, n, None)
    for kw in (dict(x=None), dict(y=None), dict(mean=None), dict(rows=0), dict(rows=-1), dict(cols=0), dict(ldx=7), dict(dtype=2), dict(dtype=-1),
               dict(eps=-1.0), dict(eps=float('nan')), dict(rows=1 << 40)):
        assert ln(**kw) == -1, kw
        assert 'layernorm_fwd' in err()
    assert ln(cols=20000, ldx=20000) == -2 and 'workspace' in err()
    need = h.lsps_layernorm_workspace_bytes(2, 20000, 0)
    assert need > 0 and ln(cols=20000, ldx=20000, ws=p, n=need - 1) == -2
    assert h.lsps_layernorm_workspace_bytes(0, 8, 0) == 0 and h.lsps_layernorm_workspace_bytes(4, 8, 7) == 0

    def lnb(dy=p, dx=p, dw=p, rows=2, cols=8, ldx=8, ldg=8, ws=None, n=0):
        return h.lsps_layernorm_bwd(dy, p, p, p, None, dx, dw, None, rows, cols, ldx, ldg, 0, ws, n, None)
    assert lnb(dy=None) == -1 and lnb(dx=None, dw=None) == -1 and lnb(ldg=7) == -1 and lnb(ldx=3) == -1
    assert lnb(rows=1000, ldx=8, ldg=8) == -2

    def ns(g=p, out=p, count=1, rows=4, cols=4, dtype=0, steps=5, abc=(3.4445, -4.775, 2.0315), eps=1e-7, ws=p, n=0):
        return h.lsps_newton_schulz(g, out, count, rows, cols, dtype, steps, *abc, eps, ws, n, None)
    for kw in (dict(g=None), dict(out=None), dict(count=0), dict(rows=0), dict(cols=-3), dict(rows=(1 << 20) + 1), dict(dtype=5), dict(steps=0),
               dict(steps=65), dict(eps=-1.0), dict(eps=float('nan')), dict(abc=(50.0, 0.0, 0.0)), dict(abc=(float('nan'), 0.0, 0.0)),
               dict(abc=(float('inf'), 0.0, 0.0)), dict(abc=(3.0, 3.0, 3.0)), dict(count=1 << 30, rows=64, cols=64)):
        assert ns(**kw) == -1, kw
        assert 'newton_schulz' in err()
    need = h.lsps_newton_schulz_workspace_bytes(1, 4, 4, 5)
    assert ns(n=need - 1) == -2 and ns(ws=None, n=need) == -2
    assert ns(ws=ctypes.c_void_p(p.value + 4), n=need) == -1 and 'aligned' in err()
    assert h.lsps_newton_schulz_workspace_bytes(0, 4, 4, 5) == 0 and h.lsps_newton_schulz_workspace_bytes(1, 4, 4, 0) == 0

    def muon(mats, lr=0.1, mu=0.9, wd=0.0, rms=0.2, gs=1.0, n=0):
        arr = (_lib.LspsMuonMatrix * max(1, len(mats)))(*mats)
        return h.lsps_muon_step(arr, len(mats), lr, mu, 1, wd, rms, gs, 5, 3.4445, -4.775, 2.0315, 1e-7, p, n, None)
    one = _lib.LspsMuonMatrix(p.value, p.value + 64, p.value + 128, 4, 4)
    assert muon([]) == -1 and muon([_lib.LspsMuonMatrix(None, p.value, p.value, 4, 4)]) == -1
    assert muon([_lib.LspsMuonMatrix(p.value, p.value, p.value, 0, 4)]) == -1
    for kw in (dict(lr=float('nan')), dict(mu=1.0), dict(mu=-0.1), dict(mu=float('nan')), dict(wd=float('inf')), dict(gs=float('nan'))):
        assert muon([one], **kw) == -1 and 'muon_step' in err(), kw
    assert muon([one]) == -2
    assert h.lsps_muon_workspace_bytes((_lib.LspsMuonMatrix * 1)(one), 1, 5) > 0 and h.lsps_muon_workspace_bytes(None, 1, 5) == 0


def test_workspace_sizes_grow_with_the_call():
    h = _lib.lib()

    def ns(*a):
        return h.lsps_newton_schulz_workspace_bytes(*a)
    assert ns(28, 256, 2304, 5) >= 28 * 4 * 2 * 256 * 2304                 # two limbs, two generations of X
    assert ns(1, 2304, 256, 5) == ns(1, 256, 2304, 5)                      # tall = wide
    assert ns(1, 256, 2304, 1) < ns(1, 256, 2304, 5) and ns(2, 100, 90, 5) > ns(1, 100, 90, 5)
    mats = (_lib.LspsMuonMatrix * 1500)(*[_lib.LspsMuonMatrix(0, 0, 0, 70, 80)] * 1500)
    one, many = h.lsps_muon_workspace_bytes(mats, 1024, 5), h.lsps_muon_workspace_bytes(mats, 1500, 5)
    assert h.lsps_muon_workspace_bytes(mats, 1, 5) < one == many            # passes share it


def test_flat_muon_sorts_parameters():
    P = torch.nn.Parameter
    for shape, want in (((4, 5), True), ((4, 3, 3, 3), True), ((5,), False), ((1, 7), False), ((7, 1, 1, 1), False), ((2, 2), True), ((), False)):
        assert optim.FlatMuon.is_matrix(P(torch.zeros(shape))) is want, shape
    opt = optim.FlatMuon([P(torch.zeros(3, 4))], lr=0.1, momentum=0.8)
    assert opt.param_groups[0]['momentum'] == 0.8 and opt.defaults['ns_steps'] == 5
    with pytest.raises(_lib.LspsHipError):
        opt.step()
    with pytest.raises(_lib.LspsHipError):
        opt.attach()


def test_configuration_keys():
    import cases
    import lsps_amd.trainers as prod
    hp = cases.hp_for('tiny')
    assert type(prod.LSPSTrainer(hp).gen_opt) is optim.FlatAdam
    tr = prod.LSPSTrainer(dict(hp, optimizer='muon', vae=dict(hp['vae'], norm='layer')))
    assert type(tr.gen_opt) is type(tr.dis_opt) is type(tr.vae_opt) is optim.FlatMuon
    keys = set(tr.vae.state_dict())
    assert {'en_fc1.model.0.weight', 'en_fc1.model.1.weight', 'en_fc1.model.1.bias', 'de_fc1.model.1.weight'} <= keys
    assert tr.vae.en_fc1.model[1].weight.shape == (hp['vae']['h_dim'],)
    with pytest.raises(ValueError):
        prod.LSPSTrainer(dict(hp, optimizer='lion'))
    with pytest.raises(ValueError):
        prod.LSPSTrainer(dict(hp, vae=dict(hp['vae'], norm='batch')))


def test_gram_chain_equals_the_iteration():
    """X (a^n I + R) built on the Gram matrix alone is n plain steps (to f64 rounding times its amplification)."""
    a, b, c = ops.NS_COEFFS
    rng = np.random.RandomState(0)
    x = rng.randn(12, 40)
    x /= np.linalg.norm(x)
    want = x
    for _ in range(3):
        k = want @ want.T
        want = a * want + (b * k + c * k @ k) @ want
    A, R, an = x @ x.T, None, 1.0
    for _ in range(3):
        S = b * A + c * A @ A
        R = S if R is None else a * R + an * S + R @ S
        T = a * A + A @ S
        A = a * T + T @ S
        an *= a
    assert np.abs(an * x + R @ x - want).max() < 1e-12


def test_two_limbs_hold_22_bits():
    rng = np.random.RandomState(1)
    v = (rng.randn(100000) * np.exp(rng.randn(100000))).astype(np.float32)
    v = v[np.abs(v) > 1e-3]
    s = np.float32(16384 / 64)
    y = v[np.abs(v) < 64] * s
    hi = y.astype(np.float16)
    lo = (y - hi.astype(np.float32)).astype(np.float16)
    off = np.abs(hi.astype(np.float64) + lo.astype(np.float64) - y.astype(np.float64))
    assert (off <= np.maximum(2.0 ** -22 * np.abs(y), 2.0 ** -25)).all()
