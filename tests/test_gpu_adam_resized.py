"""The auxiliary Adam over a parameter that is given other data, of another size, between steps: as a fresh optimizer steps it."""
import pytest
import torch

import muon_amd

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.mark.parametrize("sizes", [(20000, 300), (300, 20000)], ids=["smaller", "larger"])
def test_parameter_resized(sizes):
    gen = torch.Generator().manual_seed(0)

    def parameter(n):
        p = torch.nn.Parameter((torch.randn(n, generator=gen) * 0.05).to(DEV))
        p.grad = (torch.randn(n, generator=gen) * 1e-3).to(DEV)
        return p

    def optimizer(params):
        return muon_amd.SingleDeviceMuonWithAuxAdam([dict(params=params, use_muon=False, lr=3e-3)])

    params = [parameter(sizes[0]), parameter(70)]
    opt = optimizer(params)
    opt.step()
    other = parameter(sizes[1])
    params[0].grad = None
    params[0].data = other.detach().clone()
    params[0].grad = other.grad.clone()
    opt.state.clear()
    fresh = [other, torch.nn.Parameter(params[1].detach().clone())]
    fresh[1].grad = params[1].grad.clone()
    twin = optimizer(fresh)
    for _ in range(2):
        opt.step()
        twin.step()
        for p, q in zip(params, fresh):
            assert torch.equal(p, q)
