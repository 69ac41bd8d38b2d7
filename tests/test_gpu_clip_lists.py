"""Clipping over very many gradients."""
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
