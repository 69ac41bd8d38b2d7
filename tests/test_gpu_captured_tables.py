"""Tables that a captured HIP graph reads stay when their owners go: the cache of gradient lists, an optimizer."""
import pytest
import torch

import muon_amd
from muon_amd import _lib

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def parameters(sizes, seed=0):
    gen = torch.Generator().manual_seed(seed)
    params = [torch.nn.Parameter(torch.zeros(n, device=DEV)) for n in sizes]
    for p in params:
        p.grad = torch.randn(p.numel(), generator=gen).to(DEV)
    return params


def take_freed_memory():
    return [torch.full((2048,), 255, dtype=torch.uint8, device=DEV) for _ in range(64)]


def test_clearing_the_cache_leaves_recorded_lists():
    params = parameters([5000, 300])
    muon_amd.clip_coefficient(params, 0.1)
    before = _lib.native().tables_of_graphs()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        norm, coefficient = muon_amd.clip_coefficient(params, 0.1)
        muon_amd.clip_grad_norm_(params, 0.1)     # the same table: kept once
    assert _lib.native().tables_of_graphs() == before + 1
    muon_amd.clear_engine_cache()
    assert _lib.native().tables_of_graphs() == before + 1
    fill = take_freed_memory()
    for k in range(3):
        for i, p in enumerate(params):
            p.grad.copy_(torch.randn(p.numel(), generator=torch.Generator().manual_seed(10 * k + i)))
        grads = [p.grad.clone() for p in params]
        want = muon_amd.clip_coefficient(params, 0.1)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert float(norm) == float(want[0]) and float(coefficient) == float(want[1])
        assert all(torch.equal(p.grad, g * want[1]) for p, g in zip(params, grads))
        muon_amd.clear_engine_cache()
    assert len(fill) == 64


def test_values_of_states_outlive_the_optimizer():
    params = parameters([3000, 129])
    opt = muon_amd.AdamW(params, state_bits=8)
    opt.step()
    outs = [tuple(torch.zeros(p.numel(), dtype=torch.bfloat16, device=DEV) for _ in range(2)) for p in params]
    opt.state_values(out=outs)
    before = _lib.native().tables_of_graphs()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        opt.state_values(out=outs)
    assert _lib.native().tables_of_graphs() == before + 1
    want = [[t.clone() for t in pair] for pair in outs]
    states = [dict(opt.state[p]) for p in params]
    del opt
    fill = take_freed_memory()
    for _ in range(3):
        for pair in outs:
            for t in pair:
                t.zero_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for x, y in zip(outs, want) for a, b in zip(x, y))
    assert len(fill) == 64 and len(states) == 2
