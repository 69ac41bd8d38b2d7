"""The norm of many gradients, its coefficient and clipping in place, against sums in 64 bits.

Bounds: the norm is one rounding of a sum in 64 bits (relative 2^-24 and a few 2^-53); the coefficient two more fp32
roundings; a gradient takes one product and one rounding to its type."""
import numpy as np
import pytest
import torch

import muon_amd

gpu = pytest.mark.gpu
DEV = "cuda:0"
UNIT = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}


def make(sizes, dtypes, offset=0, std=1e-2, seed=0):
    gen = torch.Generator().manual_seed(seed)
    params = []
    for n, dtype in zip(sizes, dtypes):
        p = torch.nn.Parameter(torch.zeros(n, dtype=dtype, device=DEV))
        p.grad = (torch.randn(n + 16, generator=gen) * std).to(dtype).to(DEV)[offset:offset + n]
        params.append(p)
    return params


def check(params, max_norm, in_place):
    before = [p.grad.cpu().double() for p in params]
    norm = float(sum(g.square().sum() for g in before)) ** 0.5
    want = min(1.0, max_norm / (norm + 1e-6))
    if in_place:
        got = muon_amd.clip_grad_norm_(params, max_norm)
    else:
        got, c = muon_amd.clip_coefficient(params, max_norm)
        assert c.shape == () and c.dtype == torch.float32
        assert abs(float(c) / want - 1) <= 4 * 2.0 ** -24
    assert got.shape == () and got.dtype == torch.float32 and got.device == params[0].device
    assert abs(float(got) - norm) <= 2 * 2.0 ** -24 * norm
    for p, g in zip(params, before):
        scaled = g * (want if in_place else 1.0)
        now = p.grad.cpu().double()
        assert ((now - scaled).abs() <= (UNIT[p.dtype] + 8 * 2.0 ** -24) * scaled.abs() + 1e-40).all()
        if want == 1.0 or not in_place:
            assert torch.equal(now, g)


@gpu
@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("offset", [0, 1, 3])
@pytest.mark.parametrize("sizes", [[1], [7, 8, 9], [4095, 4096, 4097], [8191, 8192, 8193, 5], [1 << 20, 3, 70001]], ids=str)
@pytest.mark.parametrize("types", ["fp32", "bf16", "both"])
def test_norm_and_clip(types, sizes, offset, in_place):
    kinds = {"fp32": [torch.float32], "bf16": [torch.bfloat16], "both": [torch.bfloat16, torch.float32]}[types]
    params = make(sizes, [kinds[i % len(kinds)] for i in range(len(sizes))], offset)
    check(params, 1e-3, in_place)
    check(params, 1e9, in_place)


@gpu
def test_more_blocks_than_workgroups():
    params = make([8192 * 2100 + 77, 8192 * 2048], [torch.bfloat16, torch.float32])
    check(params, 0.5, False)
    check(params, 0.5, True)


@gpu
@pytest.mark.parametrize("std", [1e-30, 1e30])
def test_squares_that_fp32_does_not_hold(std):
    params = make([5000, 333], [torch.float32, torch.bfloat16], std=std)
    check(params, 1e-3 * std, False)


@gpu
def test_what_is_not_finite():
    for bad, c in ((float("inf"), 0.0), (float("nan"), float("nan"))):
        params = make([1000], [torch.float32])
        params[0].grad[17] = bad
        norm, coefficient = muon_amd.clip_coefficient(params, 1.0)
        assert np.array_equal(float(norm), bad, equal_nan=True) and np.array_equal(float(coefficient), c, equal_nan=True)
        kept = params[0].grad.clone()
        with pytest.raises(RuntimeError):
            muon_amd.clip_grad_norm_(params, 1.0, error_if_nonfinite=True)
        assert torch.equal(params[0].grad[:17], kept[:17])        # raised before anything was scaled
        muon_amd.clip_grad_norm_(params, 1.0)
        assert torch.isnan(params[0].grad[17])


@gpu
def test_strided_missing_empty_and_repeated():
    a, b, c, d = (torch.nn.Parameter(torch.zeros(n, device=DEV)) for n in ((30, 40), (5,), (0,), (6,)))
    a.grad = torch.randn(40, 30, device=DEV).t()
    c.grad = torch.zeros(0, device=DEV)
    d.grad = torch.randn(12, device=DEV)[::2]
    check([a, d], 0.3, True)
    n1 = muon_amd.clip_grad_norm_([a, b, c, d], 0.2)
    assert abs(float(n1) - 0.3) < 1e-5
    assert float(muon_amd.clip_grad_norm_(a, 0.1)) < 0.2 and float(muon_amd.clip_grad_norm_(iter([b]), 1.0)) == 0.0
    assert [float(t) for t in muon_amd.clip_coefficient([b], 1.0)] == [0.0, 1.0]
    with pytest.raises(ValueError):
        muon_amd.clip_grad_norm_([a, a], 1.0)
    zero = torch.nn.Parameter(torch.zeros(3, device=DEV))
    zero.grad = torch.zeros(3, device=DEV)
    check([zero], 1.0, True)
    check([d], 0.0, True)


@gpu
def test_coefficient_feeds_the_step():
    params, twins = (make([5000, 300], [torch.float32] * 2) for _ in range(2))
    opts = [muon_amd.AdamW(ps, lr=1e-2) for ps in (params, twins)]
    _, c = muon_amd.clip_coefficient(params, 0.1)
    opts[0].step(grad_scale=c)
    muon_amd.clip_grad_norm_(twins, 0.1)
    opts[1].step()
    for p, q in zip(params, twins):
        assert torch.equal(p, q)


@gpu
def test_streams_and_repeats():
    params = make([300000, 77], [torch.bfloat16, torch.float32])
    first = [muon_amd.clip_coefficient(params, 1.0) for _ in range(3)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        first.append(muon_amd.clip_coefficient(params, 1.0))
    torch.cuda.synchronize()
    assert len({(float(n), float(c)) for n, c in first}) == 1     # the same bits each time, each in memory of its own


def test_refusals():
    p = torch.nn.Parameter(torch.zeros(3))
    p.grad = torch.zeros(3)
    with pytest.raises(muon_amd.MuonAmdError):
        muon_amd.clip_grad_norm_([p], 1.0)
    with pytest.raises(ValueError):
        muon_amd.clip_grad_norm_([p], -1.0)
    with pytest.raises(ValueError):
        muon_amd.clip_coefficient([p], float("nan"))
    p.grad = None
    assert float(muon_amd.clip_grad_norm_([p], 1.0)) == 0.0 and float(muon_amd.clip_grad_norm_([], 1.0)) == 0.0


def test_tables_are_checked():
    from muon_amd import _lib, plan
    lib = _lib.load()
    d = np.zeros(1, dtype=_lib.GRAD_DESC)
    d["grad"], d["numel"] = 4096, 10000
    prefix = plan.adam_block_prefix([10000])
    assert lib.muon_amd_validate_grads(_lib.host_ptr(d), 1, _lib.host_ptr(prefix)) == 0
    assert lib.muon_amd_validate_grads(_lib.host_ptr(d), 1, _lib.host_ptr(np.array([0, 1], dtype=np.int32))) == -1
    for name, value in (("grad", 0), ("grad", 4098), ("numel", 0), ("dtype", 3)):
        bad = d.copy()
        bad[name] = value
        assert lib.muon_amd_validate_grads(_lib.host_ptr(bad), 1, _lib.host_ptr(prefix)) == -1
    assert lib.muon_amd_grad_norm(None, None, 1, 1, None, 1.0, None, None) == -1


@gpu
def test_captured_calls():
    """Recorded into a graph, both calls read the gradients as they are at each replay; a list that no call has seen
    cannot be recorded; other lists do not take the recorded one's table away."""
    params = make([5000, 300], [torch.float32, torch.bfloat16])
    other = make([77], [torch.float32])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        muon_amd.clip_coefficient(params, 0.1)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        norm, coefficient = muon_amd.clip_coefficient(params, 0.1)
        with pytest.raises(muon_amd.MuonAmdError):
            muon_amd.clip_coefficient(other, 0.1)
        muon_amd.clip_grad_norm_(params, 0.1)
    for _ in range(40):                                           # more lists than are kept
        muon_amd.clip_coefficient(make([50], [torch.float32]), 1.0)
    for k in range(4):
        for i, p in enumerate(params):
            p.grad.copy_(torch.randn(p.numel(), generator=torch.Generator().manual_seed(10 * k + i)) * (k + 1))
        before = [p.grad.clone() for p in params]
        want = muon_amd.clip_coefficient(params, 0.1)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert float(norm) == float(want[0]) and float(coefficient) == float(want[1])
        for p, g in zip(params, before):
            assert torch.equal(p.grad, (g.float() * want[1]).to(g.dtype))


@gpu
def test_gradients_that_share_memory():
    params = make([1000, 1000, 500], [torch.float32] * 3)
    params[1].grad = params[0].grad                               # counted twice by the norm; scaled twice it would be a race
    check(params, 1e-3, False)
    for other in (params[0].grad, params[0].grad[250:750]):
        params[2 if other.numel() == 500 else 1].grad = other
        before = [p.grad.clone() for p in params]
        with pytest.raises(ValueError, match="share memory"):
            muon_amd.clip_grad_norm_(params, 1e-3)
        assert all(torch.equal(p.grad, g) for p, g in zip(params, before))
        params[1].grad = params[0].grad.clone()
    whole = torch.full((1500,), 0.5, device=DEV)                  # views of one buffer that lie next to each other
    params[0].grad, params[2].grad = whole[:1000], whole[1000:]
    check(params, 1e-3, True)
