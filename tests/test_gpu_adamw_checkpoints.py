"""Checkpoints of torch.optim.AdamW loaded into muon_amd.AdamW."""
import copy

import pytest
import torch

import muon_amd

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def trained(dtype, **options):
    gen = torch.Generator().manual_seed(0)
    params = [torch.nn.Parameter((torch.randn(*s, generator=gen) * 0.05).to(dtype).to(DEV)) for s in ((300,), (33, 65))]
    params.append(torch.nn.Parameter((torch.randn(20, 30, generator=gen) * 0.05).to(dtype).to(DEV).t()))      # its states are strided alike
    opt = torch.optim.AdamW(params, lr=3e-3, betas=(0.9, 0.95), weight_decay=0.01, foreach=False, **options)
    for _ in range(2):
        for p in params:
            p.grad = (torch.randn(p.shape, generator=gen) * 1e-3).to(dtype).to(DEV)
        opt.step()
    return params, opt


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_states_are_widened(dtype):
    params, old = trained(dtype)
    new = muon_amd.AdamW(params, state_bits=32)
    saved = copy.deepcopy(old.state_dict())
    new.load_state_dict(saved)
    before = [p.detach().double() for p in params]
    states = [{k: old.state[p][k].double() for k in ("exp_avg", "exp_avg_sq")} for p in params]
    assert all(old.state[p]["exp_avg"].dtype == dtype for p in params)
    new.step()
    for p, p0, s in zip(params, before, states):
        g = p.grad.double()
        m, v = 0.9 * s["exp_avg"] + 0.1 * g, 0.95 * s["exp_avg_sq"] + 0.05 * g * g
        for k, want in (("exp_avg", m), ("exp_avg_sq", v)):
            assert new.state[p][k].dtype == torch.float32
            torch.testing.assert_close(new.state[p][k].double(), want, rtol=1e-5, atol=1e-12)
        want = p0 * (1 - 3e-3 * 0.01) - 3e-3 / (1 - 0.9 ** 3) * m / ((v / (1 - 0.95 ** 3)).sqrt() + 1e-8)
        torch.testing.assert_close(p.detach().double(), want, rtol=2.0 ** -8 if dtype == torch.bfloat16 else 1e-6, atol=1e-8)
        assert new.state[p]["step"] == 3


def test_states_of_8_bits_are_not_made_from_others():
    params, old = trained(torch.bfloat16)
    new = muon_amd.AdamW(params, state_bits=8)
    new.load_state_dict(old.state_dict())
    with pytest.raises(NotImplementedError):
        new.step()


@pytest.mark.parametrize("option", ["amsgrad", "maximize"])
def test_other_algorithms_are_refused(option):
    params, old = trained(torch.float32, **{option: True})
    for new in (muon_amd.AdamW(params), muon_amd.AdamW(params, state_bits=8)):
        with pytest.raises(NotImplementedError, match=option):
            new.load_state_dict(old.state_dict())
        assert not new.state and new.param_groups[0]["lr"] == 1e-3
