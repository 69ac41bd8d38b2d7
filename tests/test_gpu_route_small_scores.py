"""Routing by scores near and below the smallest number of 32 bits, against the formulas in 64 bits (GPU): the weights of a token's choices are ratios
of their scores, and its shares of the balance loss ratios too, which are ordinary numbers where the scores are not.  Bounds as in test_gpu_route_scored.py, for
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
@pytest.mark.parametrize("normalize", [True, False])
@pytest.mark.parametrize("experts,k,groups,kept", [(8, 2, 1, 1), (16, 4, 4, 2), (48, 6, 6, 3), (64, 32, 1, 1), (256, 8, 8, 4), (1024, 32, 16, 5)])
def test_sigmoids_that_vanish(experts, k, groups, kept, normalize, dtype):
    """All of a token's sigmoids at e^-60 to e^-300, between tokens of ordinary ones."""
    logits, mask, dw, bias = make((120, experts), k, dtype, seed=experts, masked=True)
    logits[::2] = (logits[::2].float() * 3 - torch.linspace(60, 300, 60)[:, None]).to(dtype)
    for b in (None, torch.zeros(experts)):
        r, _ = check(logits, mask, dw, b, k, "sigmoid", groups, kept, normalize)
        if normalize:                                            # k numbers of 32 bits that add up to one
            assert ((r.weights.sum(1) - 1).abs()[mask.to(DEV)] <= 3 * k * U).all()


@gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("experts,k", [(8, 4), (64, 8), (256, 32)])
def test_choices_far_below_the_first(experts, k, dtype):
    """A token's choices reach from an ordinary score to ones that vanish, and to weights that do not (from -20 to -100: e^-80)."""
    g = torch.Generator().manual_seed(k)
    logits = torch.full((64, experts), -150.0)
    logits[:, :k] = -torch.linspace(0, 80, k) - torch.linspace(-30, 30, 64)[:, None] + torch.rand(64, k, generator=g)
    logits = logits[:, torch.randperm(experts, generator=g)].to(dtype)
    dw = torch.randn(64, k, generator=g)
    for scores in ("sigmoid", "softmax"):
        check(logits, None, dw, None, k, scores)


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


@gpu
def test_a_row_that_is_no_number_far_down():
    """NaN and infinities among choices far down stay what they are in other rows: no number for the row, nothing for its neighbours."""
    logits, _, dw, _ = make((64, 16), 4, F32, std=30.0)
    logits -= 100
    clean, _ = check(logits, None, dw, None, 4, "sigmoid")
    logits[7, 2] = float("nan")
    logits[9, 5] = INF
    r = muon_amd.route_topk(logits.to(DEV), 4, scores="sigmoid")
    rest = torch.tensor([i for i in range(64) if i not in (7, 9)])
    assert torch.equal(r.weights[rest], clean.weights[rest]) and torch.equal(r.indices[rest], clean.indices[rest])
    assert torch.isnan(r.weights[7]).any() and r.weights[9, 0] == 1 and r.indices[9, 0] == 5


@gpu
@pytest.mark.parametrize("scores", ["softmax", "sigmoid"])
@pytest.mark.parametrize("experts,groups,kept", [(8, 4, 2), (16, 4, 2), (60, 10, 5), (64, 8, 4), (256, 32, 16)])
def test_groups_at_the_smallest_number(experts, groups, kept, scores):
    """Groups whose scores are sums of numbers on both sides of 2^-126, where the smaller ones are flushed: chosen as in 64 bits."""
    g = torch.Generator().manual_seed(experts)
    logits = -85.5 - 6.5 * torch.rand(3000, experts, generator=g)
    if scores == "softmax":
        logits = logits - logits.amax(1, keepdim=True) - 85.5 - torch.rand(3000, 1, generator=g)
        logits[:, 0] = 0.0
    dw = torch.randn(3000, 1, generator=g)
    for k in (1, kept):
        check(logits, None, dw.expand(3000, k), None, k, scores, groups, kept)
