"""AdamW with 8-bit states and NaN of any bits."""
import pytest
import torch

import muon_amd

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
F32, BF16 = torch.float32, torch.bfloat16
PATTERNS = [(F32, 0xFFFFFFFF), (F32, 0xFFF00001), (F32, 0xFFF00002), (F32, 0x7FFFFFFF), (F32, 0x7F800001), (F32, 0xFF800001),
            (BF16, 0xFFFF), (BF16, 0xFFF1), (BF16, 0xFFF0), (BF16, 0x7FFF), (BF16, 0x7F81), (BF16, 0xFF81)]


@pytest.mark.parametrize("dtype,bits_of_nan", PATTERNS, ids=lambda v: f"{v:X}" if isinstance(v, int) else str(v)[6:])
def test_nan_of_any_bits_shows_in_its_block(dtype, bits_of_nan):
    p = torch.nn.Parameter(torch.zeros(1000, dtype=dtype, device=DEV))
    p.grad = (torch.randn(1000, generator=torch.Generator().manual_seed(1)) * 1e-3).to(dtype).to(DEV)
    integers = p.grad.view(torch.int32 if dtype == F32 else torch.int16)
    integers[300] = bits_of_nan - (1 << (32 if dtype == F32 else 16)) * (bits_of_nan >> (31 if dtype == F32 else 15))
    p.grad[301] = 1e4                             # far larger than the rest of the block, in the same lane
    opt = muon_amd.AdamW([p], lr=1e-3, state_bits=8)
    inside = (torch.arange(1000, device=DEV) >= 256) & (torch.arange(1000, device=DEV) < 384)
    for _ in range(2):
        opt.step()
        p.grad.fill_(1e-3)
        m, v = opt.state_values()[0]
        assert torch.equal(torch.isnan(m), inside) and torch.equal(torch.isnan(v), inside)
        assert all((opt.state[p][k][2] == 255) and (opt.state[p][k] != 255).sum() == 7 for k in ("exp_avg_exponent", "exp_avg_sq_exponent"))
    assert torch.equal(torch.isnan(p.detach()), inside)
