"""AdamW over parameters that share memory: refused before anything is stepped."""
import pytest
import torch

import muon_amd

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def with_gradient(t):
    p = torch.nn.Parameter(t)
    p.grad = torch.ones_like(t)
    return p


@pytest.mark.filterwarnings("ignore:optimizer contains a parameter group with duplicate parameters")
@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_shared_parameters(dtype, bits):
    whole = torch.full((3000,), 0.5, dtype=dtype, device=DEV)
    p = with_gradient(whole[:1000])
    for others in ([p], [with_gradient(whole[:1000])], [with_gradient(whole[1000:2000]), with_gradient(whole[999:1003])],
                   [with_gradient(torch.zeros(70, dtype=dtype, device=DEV)), with_gradient(whole[500:600])]):
        opt = muon_amd.AdamW([p, *others], lr=0.1, state_bits=bits)
        with pytest.raises(ValueError, match="share memory"):
            opt.step()
        assert (whole == 0.5).all() and all(opt.state[q]["step"] == 0 and not opt.state[q]["exp_avg"].any() for q in (p, *others))


@pytest.mark.parametrize("bits", [32, 8])
def test_neighbours_in_one_buffer(bits):
    whole = torch.full((3000,), 0.5, device=DEV)
    opt = muon_amd.AdamW([with_gradient(t) for t in (whole[1000:1001], whole[:1000], whole[1001:])], lr=0.1, state_bits=bits)
    opt.step()                                    # (from here on states of 8 bits differ by their places' dither)
    assert len(whole.unique()) == 1 and float(whole[0]) < 0.45
