"""Routing by scores near and below the smallest number of 32 bits, against the formulas in 64 bits (GPU): the weights of a token's choices are ratios
of their scores, which are ordinary numbers where the scores are not.  Bounds as in test_gpu_route_scored.py, for
every row; the balance loss has E 2^-126 more: E sum_e (counts_e / n k) (mean share_e), where the factors of the shares add up to one, and a share below 2^-126 may
be zero (an expert that has a token's whole probability and none of its choices leaves a balance loss of e^-200: there is no such number in 32 bits)."""
import pytest
import torch

import muon_amd
from test_gpu_route_scored import BF16, DEV, F32, INF, U, UNIT, exact, make

gpu = pytest.mark.gpu


def check(logits, mask, dw, bias, k, scores, groups=1, kept=1, normalize=True, cb=0.3, cz=0.02):
    leaf = logits.to(DEV).requires_grad_()
    m, b = (None if t is None else t.to(DEV) for t in (mask, bias))
    r = muon_amd.route_topk(leaf, k, mask=m, normalize=normalize, scores=scores, bias=b, groups=groups, groups_kept=kept)
    grad, = torch.autograd.grad((r.weights, r.balance_loss, r.z_loss), leaf, (dw.to(DEV), torch.tensor(cb, device=DEV), torch.tensor(cz, device=DEV)))
    want = exact(logits, k, scores, bias, groups, kept, mask, normalize, dw, cb, cz)
    T, E = logits.shape
    assert torch.equal(r.indices.cpu().long(), want["indices"]) and torch.equal(r.counts.cpu().long(), want["counts"])
    assert ((r.weights.detach().cpu().double() - want["weights"]).abs() <= 128 * U * want["weights"] + 1e-37).all()
    sums = (T / 64 + 256) * U
    assert abs(float(r.balance_loss.detach()) - want["balance"]) <= sums * want["balance"] + E * 2.0 ** -126
    assert abs(float(r.z_loss.detach()) - want["z"]) <= (sums + 4 * U) * want["z"] + 128 * U * float(want["lse"].abs().max())
    off = (grad.cpu().double() - want["grad"]).abs() - 256 * U * want["mag"] - UNIT[logits.dtype] * want["grad"].abs()
    assert off.max() <= 1e-37
    return r, grad


@gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("below", [80, 88, 95, 200])
@pytest.mark.parametrize("experts,k,groups,kept", [(8, 2, 1, 1), (32, 4, 4, 2), (64, 32, 1, 1), (256, 8, 8, 4)])
def test_an_expert_that_is_not_available_far_above_the_others(experts, k, groups, kept, below, dtype):
    """Softmax: what the token may choose from has next to nothing of its probability, and the weights of two numbers all the same."""
    logits, mask, dw, bias = make((80, experts), k, dtype, seed=below, masked=True)
    logits[:, 3] = below
    for low in (-INF, -2.0, torch.finfo(F32).min):
        b = torch.zeros(experts)
        b[3] = low
        r, _ = check(logits, mask, dw, b, k, "softmax", groups, kept)
        assert ((r.weights.sum(1) - 1).abs()[mask.to(DEV)] <= 3 * k * U).all()
        check(logits, mask, dw, b, k, "softmax", groups, kept, normalize=False)
