"""linear_cross_entropy where logits are far from zero (GPU): loss and logsumexp each against its own bound.

All logits of a token are one number x, so the loss is ln V whatever x, and lse is x + ln V.  With U = 2^-24 the logarithm is held to 200 U of itself as in
test_gpu_head.py (the sum of V equal terms, a logarithm in base 2, a product); x enters the loss as a difference of two equal numbers, and lse is rounded once (U of itself)."""
import math

import pytest
import torch

import muon_amd

DEV = "cuda:0"
U = 2.0 ** -24
BF16 = torch.bfloat16


@pytest.mark.gpu
@pytest.mark.parametrize("tokens", [1, 10, 40, 140, 700])
@pytest.mark.parametrize("at", [0.0, 1.0, 1e4, -1e4, 3e7, -3e30])
def test_loss_and_logsumexp(at, tokens):
    v, d = 1000, 64
    h, w = torch.zeros(tokens, d, dtype=BF16), torch.zeros(v, d, dtype=BF16)
    h[:, 0], w[:, 0] = at, 1.0
    t = (torch.arange(tokens) * 37) % v
    x = float(h[0, 0])
    each = muon_amd.linear_cross_entropy(h.to(DEV), w.to(DEV), t.to(DEV), reduction="none")
    assert ((each.loss.double().cpu() - math.log(v)).abs() <= 200 * U * math.log(v)).all()
    assert ((each.lse.double().cpu() - (x + math.log(v))).abs() <= 200 * U * math.log(v) + U * abs(x + math.log(v))).all()
    for reduction, n in (("sum", tokens), ("mean", 1)):
        out = muon_amd.linear_cross_entropy(h.to(DEV).requires_grad_(), w.to(DEV), t.to(DEV), reduction=reduction)
        # (sums of up to 700 numbers in fp32, at most 64 one after the other: 64 U more)
        assert abs(float(out.loss.detach()) - n * math.log(v)) <= n * 264 * U * math.log(v)
        assert torch.equal(out.lse.detach(), each.lse)
