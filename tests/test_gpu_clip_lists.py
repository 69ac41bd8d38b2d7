"""Clipping over very many gradients, and over gradients that cannot be written."""
import pytest
import torch

import muon_amd

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def test_more_gradients_than_two_steps_of_the_lookup_cover():
    """A wave looks 64 entries at a time up in a table of 64^3 and more tensors."""
    n = 64 ** 3 + 64 ** 2 + 700
    flat = torch.ones(n, device=DEV)
    param = torch.zeros(1, device=DEV)
    params = []
    for g in flat.split(1):
        p = torch.nn.Parameter(param)
        p.grad = g
        params.append(p)
    norm = muon_amd.clip_grad_norm_(params, 0.5 * n ** 0.5)
    assert abs(float(norm) - n ** 0.5) <= 1e-6 * n ** 0.5
    assert float(flat.min()) == float(flat.max()) and abs(float(flat.max()) - 0.5) < 1e-6


def test_a_broadcast_gradient_is_refused_before_anything_is_scaled():
    a, b = (torch.nn.Parameter(torch.zeros(5, 6, device=DEV)) for _ in range(2))
    a.grad = torch.ones(5, 6, device=DEV)
    b.grad = torch.ones(6, device=DEV).expand(5, 6)
    norm, _ = muon_amd.clip_coefficient([a, b], 1.0)              # (reading it is fine)
    assert abs(float(norm) - 60 ** 0.5) < 1e-5
    with pytest.raises(ValueError, match="share memory"):
        muon_amd.clip_grad_norm_([a, b], 1.0)
    assert (a.grad == 1).all() and (b.grad == 1).all()
