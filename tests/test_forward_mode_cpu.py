"""Forward-mode derivatives (torch.autograd.forward_ad) of layer norm, Newton-Schulz and the Muon step: refused, not dropped."""
import pytest
import torch
from torch.autograd import forward_ad

from lsps_amd import _lib, ops


def test_dual_tensors_are_refused():
    x, w = torch.randn(3, 4), torch.ones(4)
    with forward_ad.dual_level():
        xd, wd = forward_ad.make_dual(x, torch.ones_like(x)), forward_ad.make_dual(w, torch.ones_like(w))
        param = torch.nn.Parameter(w.clone())
        for call in (lambda: ops.layer_norm(xd, 4), lambda: ops.layer_norm(xd, 4, param), lambda: ops.layer_norm(x, 4, wd),
                     lambda: ops.layer_norm(x, 4, w, wd), lambda: ops.newton_schulz(xd),
                     lambda: ops.muon_step_([x.clone()], [xd], [x.clone()], lr=0.1), lambda: ops.muon_step_([xd], [x], [x.clone()], lr=0.1)):
            with pytest.raises(_lib.LspsHipError, match='forward-mode'):
                call()
        for call in (lambda: ops.layer_norm(x, 4, w), lambda: ops.newton_schulz(x)):      # no tangent: as ever (here: no CPU path)
            with pytest.raises(_lib.LspsHipError, match='HIP'):
                call()
