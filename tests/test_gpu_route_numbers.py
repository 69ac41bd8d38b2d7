"""route_topk where its numbers are large, or not there: logits far from zero, whole rows of a type's lowest value, and upstream
gradients that mean nothing.  Bounds as in test_gpu_route: they go by differences of logits, not by their size."""
import pytest
import torch

import muon_amd
from test_gpu_route import BF16, DEV, F32, U, UNIT, exact, make

pytestmark = pytest.mark.gpu


def parts(logits, k, mask, dw, normalize=True):
    """Gradients of the weights and of the balance loss against 64 bits."""
    for names in (["weights"], ["balance_loss"], ["weights", "balance_loss"]):
        leaf = logits.to(DEV).requires_grad_()
        r = muon_amd.route_topk(leaf, k, mask=None if mask is None else mask.to(DEV), normalize=normalize)
        give = {"weights": dw.to(DEV), "balance_loss": torch.tensor(0.3, device=DEV)}
        got, = torch.autograd.grad([getattr(r, n) for n in names], leaf, [give[n] for n in names])
        want = exact(logits, k, mask, normalize, dw if "weights" in names else 0 * dw, 0.3 if "balance_loss" in names else 0.0, 0.0)
        assert torch.equal(r.indices.cpu().long().reshape(want["indices"].shape), want["indices"])
        assert ((r.weights.detach().cpu().double() - want["weights"]).abs() <= 128 * U * want["weights"] + 1e-37).all()
        off = (got.cpu().double() - want["grad"]).abs() - 256 * U * want["mag"] - UNIT[logits.dtype] * want["grad"].abs()
        assert off.max() <= 1e-37, (names, float(off.max()))


@pytest.mark.parametrize("normalize", [True, False])
@pytest.mark.parametrize("experts,k", [(8, 2), (48, 6), (200, 8), (1000, 20)])
@pytest.mark.parametrize("shift", [1e2, -3e3, 1e5, -1e7, 1e30])
def test_logits_far_from_zero(shift, experts, k, normalize):
    logits, mask, dw = make((60, experts), k, F32, seed=experts, masked=True)
    parts(logits + shift, k, mask, dw, normalize)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("experts,k", [(8, 2), (48, 6), (300, 8)])
def test_rows_of_the_lowest_value(experts, k, dtype):
    logits, _, dw = make((40, experts), k, dtype, seed=3)
    logits[5] = torch.finfo(dtype).min
    logits[9] = torch.finfo(dtype).min
    logits[9, 3] = -float("inf")
    logits[11] = torch.finfo(dtype).max
    logits[13, 1:] = torch.finfo(dtype).min
    for normalize in (True, False):
        parts(logits, k, None, dw, normalize)


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
