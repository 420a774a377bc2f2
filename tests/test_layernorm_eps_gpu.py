"""Layer norm with an `eps` that counts (csrc/layernorm.hip), forward and backward, at every variant's width; the formula and the
tolerances are those of test_layernorm_gpu.py."""
import pytest
import torch

from test_layernorm_gpu import check_backward, check_forward, make

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('eps', [1e-3, 0.1, 1.0, 30.0])
@pytest.mark.parametrize('rows,cols', [(5, 3), (64, 50), (130, 128), (100, 257), (7, 1023), (41, 2049), (9, 8192), (2, 16384), (3, 20001)])
def test_eps(rows, cols, dtype, eps):
    from lsps_amd import ops
    x, dy, w, b = make(rows, cols, dtype)
    x = x * 0.1 if cols % 2 else x                           # also where the variance is far below eps
    for t in (x, w, b):
        t.requires_grad_(True)
    y = ops.layer_norm(x, cols, w, b, eps)
    check_forward(y.detach(), x.detach(), w.detach(), b.detach(), eps)
    dx, dw, db = torch.autograd.grad(y, (x, w, b), dy)
    check_backward(dx, dw, db, x.detach(), dy, w.detach(), b.detach(), eps)
    assert torch.equal(ops.layer_norm(x.detach(), cols, w.detach(), b.detach(), eps), y)


@pytest.mark.parametrize('cols', [50, 700, 3000, 18000])
def test_constant_rows(cols):
    """No variance: eps alone under the root, the result is the bias; zero eps there is 0 / 0."""
    from lsps_amd import ops
    x = torch.full((4, cols), 2.0, device='cuda')
    w, b = torch.full((cols,), 3.0, device='cuda'), torch.randn(cols, device='cuda')
    assert torch.equal(ops.layer_norm(x, cols, w, b, 0.25), b.expand(4, cols))
    assert bool(torch.isnan(ops.layer_norm(x, cols, w, b, 0.0)).all())
