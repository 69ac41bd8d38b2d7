"""AdamW where numbers end: NaN of any bits, and second moments that only subnormal numbers hold, with eps = 0.

Bounds.  U = 2^-24.  With eps = 0 a first step from zeros gives m / sqrt(v) = w1 g / (sqrt(w2) |g|) whatever g is.  v is a
product and a fused product and sum in fp32: within 2^-149 for each of the two roundings where it is subnormal, and 2 U of
itself else; the root halves what that is relative to v.  m takes 2 U, root, quotient and products together 16 U."""
import numpy as np
import pytest
import torch

import muon_amd

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
U = 2.0 ** -24
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


@pytest.mark.parametrize("eps", [0.0, 1e-30, 1e-20])
@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_second_moments_below_the_normal_numbers(dtype, bits, eps):
    lr, betas = 2.0 ** -7, (0.9, 0.95)
    sign = torch.where(torch.arange(3000) % 2 == 0, 1.0, -1.0)
    g = (sign * torch.logspace(-21, -17, 3000)).to(dtype)
    p = torch.nn.Parameter(torch.zeros(3000, dtype=dtype, device=DEV))
    p.grad = g.to(DEV)
    opt = muon_amd.AdamW([p], lr=lr, betas=betas, eps=eps, weight_decay=0.0, state_bits=bits)
    opt.step()
    g = g.double().numpy()
    w1, w2 = (float(np.float32(1 - b)) for b in betas)
    v = w2 * g * g
    d = np.sqrt(v / (1 - betas[1])) + eps
    want = -lr / (1 - betas[0]) * w1 * g / d
    slack = 18 * U + 0.5 * (2 * U + 2 * 2.0 ** -149 / v)
    got = p.detach().cpu().double().numpy()
    assert np.isfinite(got).all()
    # (from the root's slope: 0.5 of v's slack while that is small, at most all of it)
    allowed = np.abs(want) * (2 * slack + (U if dtype == F32 else 2.0 ** -8))
    np.testing.assert_array_less(np.abs(got - want)[v > 2.0 ** -145], allowed[v > 2.0 ** -145])
