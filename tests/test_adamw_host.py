"""AdamW without a GPU: every way to step says so in the package's own error."""
import pytest
import torch

import muon_amd


@pytest.mark.parametrize("use_graph", [False, True])
@pytest.mark.parametrize("bits", [32, 8])
def test_parameters_on_the_host(bits, use_graph):
    p = torch.nn.Parameter(torch.zeros(10))
    p.grad = torch.zeros(10)
    opt = muon_amd.AdamW([p], state_bits=bits, use_graph=use_graph)
    with pytest.raises(muon_amd.MuonAmdError, match="no CPU implementation"):
        opt.step()
    assert not opt.state[p]
