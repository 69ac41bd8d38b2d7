"""The gate of residual_norm in fp32, far on its low side: relative to itself.

h = sigmoid(z) / sqrt(1 + eps) over rows of ones with x = 0.  The sigmoid is within 8 U of itself, the norm's factor within 4
U, two products 2 U, h's rounding 1: 15 U, while sigmoid(z) is a normal number."""
import numpy as np
import pytest
import torch

import muon_amd

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.mark.parametrize("kind", ["channel", "token"])
def test_low_side(kind):
    z = torch.linspace(-86, 12, 4096)
    shape = (1, 4096) if kind == "channel" else (4096, 4)
    gate = (z[None] if kind == "channel" else z[:, None]).to(DEV).requires_grad_()
    x, one = torch.zeros(shape, device=DEV), torch.ones(shape, device=DEV)
    w = torch.ones(shape[1], device=DEV)
    h, y = muon_amd.residual_norm(x, one, w, w, gate=gate)
    want = 1 / (1 + np.exp(-z.double().numpy())) / np.sqrt(1 + float(np.float32(1e-6)))
    got = h.detach().cpu().double().numpy()
    got = got[0] if kind == "channel" else got[:, 0]
    assert (np.abs(got - want) <= 15 * 2.0 ** -24 * want).all(), float((np.abs(got / want - 1) * 2 ** 24).max())
    # dz = dh nb sig (1 - sig): 1 - sig has the rounding of sig near one, U of one
    dz, = torch.autograd.grad(h, gate, torch.ones_like(h))
    n = 1 if kind == "channel" else 4
    sig = 1 / (1 + np.exp(-z.double().numpy()))
    exact = n * sig * (1 - sig) / np.sqrt(1 + float(np.float32(1e-6)))
    off = np.abs(dz.cpu().double().numpy().ravel() - exact)
    assert (off <= 24 * 2.0 ** -24 * exact + 8 * 2.0 ** -24 * n * sig * sig).all()
