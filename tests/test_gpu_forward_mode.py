"""Forward-mode derivatives: residual_norm and route_topk have none, and say so instead of dropping the tangent."""
import pytest
import torch
import torch.autograd.forward_ad as fwd

import muon_amd

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.mark.parametrize("leaf", [False, True], ids=["constant", "requires-grad"])
@pytest.mark.parametrize("name", ["x", "block", "post_weight", "pre_weight", "gate", "scale"])
def test_residual_norm(name, leaf):
    t = {n: torch.randn(*s, device=DEV) for n, s in dict(x=(3, 8), block=(3, 8), post_weight=(8,), pre_weight=(8,), gate=(3, 8), scale=(8,)).items()}
    with fwd.dual_level():
        t[name] = fwd.make_dual(t[name].requires_grad_(leaf), torch.ones_like(t[name]))
        with pytest.raises(NotImplementedError, match="forward-mode"):
            muon_amd.residual_norm(**t)
        with torch.no_grad(), pytest.raises(NotImplementedError, match="forward-mode"):
            muon_amd.residual_norm(**t)
        primal = {n: fwd.unpack_dual(v).primal for n, v in t.items()}
        muon_amd.residual_norm(**primal)


@pytest.mark.parametrize("leaf", [False, True], ids=["constant", "requires-grad"])
def test_route_topk(leaf):
    z = torch.randn(4, 8, device=DEV).requires_grad_(leaf)
    with fwd.dual_level():
        dual = fwd.make_dual(z, torch.ones_like(z))
        with pytest.raises(NotImplementedError, match="forward-mode"):
            muon_amd.route_topk(dual, 2)
        muon_amd.route_topk(fwd.unpack_dual(dual).primal, 2)
