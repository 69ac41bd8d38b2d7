"""route_topk and upstream gradients that mean nothing."""
import pytest
import torch

import muon_amd
from test_gpu_route import DEV, F32, make

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("normalize", [True, False])
@pytest.mark.parametrize("experts,k", [(8, 4), (48, 6), (300, 8), (1024, 32), (5, 5)])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")], ids=["nan", "inf"])
def test_gradients_of_choices_that_are_not_there(bad, experts, k, normalize):
    """A weight whose index is -1 is the constant zero: whatever arrives for it, nothing flows on."""
    logits, mask, dw = make((50, experts), k, F32, seed=experts, masked=True)
    logits[7, 2:] = -float("inf")                 # two experts for k choices
    logits[8] = -float("inf")
    logits[10, 1:] = -float("inf")
    mask[[7, 10]] = True
    leaf = logits.to(DEV).requires_grad_()
    r = muon_amd.route_topk(leaf, k, mask=mask.to(DEV), normalize=normalize)
    clean, = torch.autograd.grad(r.weights, leaf, dw.to(DEV), retain_graph=True)
    dirty = dw.masked_fill(r.indices.cpu() < 0, bad)
    got, = torch.autograd.grad(r.weights, leaf, dirty.to(DEV))
    assert torch.isfinite(clean).all() and torch.equal(got, clean)
