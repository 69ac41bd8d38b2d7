"""AdamW.step inside a HIP graph that the program captures: only over tensors that a step has seen; a replay is that step
again, whatever eager steps do in between."""
import pytest
import torch

import muon_amd
from test_gpu_adamw import BETAS, EPS, LR, WD, make

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
F32, BF16 = torch.float32, torch.bfloat16


def optimizer(params, bits, **options):
    return muon_amd.AdamW(params, lr=LR, betas=BETAS, eps=EPS, weight_decay=WD, state_bits=bits, **options)


def twin_of(opt, params, bits, step):
    """An optimizer of its own over copies, `step` steps old."""
    copies = [torch.nn.Parameter(p.detach().clone()) for p in params]
    other = optimizer(copies, bits)
    for q, p in zip(copies, params):
        q.grad = p.grad.clone()
        other.state[q].update({k: v.clone() if isinstance(v, torch.Tensor) else v for k, v in opt.state[p].items()}, step=step)
    return other, copies


def same(opt, params, other, copies):
    for p, q in zip(params, copies):
        assert torch.equal(p, q)
        for k, v in opt.state[p].items():
            assert not isinstance(v, torch.Tensor) or torch.equal(v, other.state[q][k])


@pytest.mark.parametrize("bits", [32, 8])
def test_captured_steps(bits):
    params = make([5000, (129, 65)], F32) + make([300], BF16)
    opt = optimizer(params, bits)
    scale = torch.full((), 0.5, device=DEV)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        opt.step(grad_scale=scale)                # the one step that a capture needs before it
    torch.cuda.current_stream().wait_stream(side)
    stranger = make([77], F32)
    unseen = optimizer(stranger, bits)
    recorded = [p.grad for p in params]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        opt.step(grad_scale=scale)
        with pytest.raises(muon_amd.MuonAmdError, match="captured"):
            unseen.step()
        params[0].grad = torch.zeros_like(params[0])
        with pytest.raises(muon_amd.MuonAmdError, match="captured"):
            opt.step(grad_scale=scale)            # a gradient at an address that no step has seen
        params[0].grad = recorded[0]
        params[1].grad = None
        with pytest.raises(muon_amd.MuonAmdError, match="captured"):
            opt.step(grad_scale=scale)            # another list
        params[1].grad = recorded[1]
    assert all(opt.state[p]["step"] == 2 for p in params) and not unseen.state[stranger[0]]
    unseen.step()                                 # what was refused works outside
    for k in range(5):
        for i, g in enumerate(recorded):
            g.copy_(torch.randn(g.shape, generator=torch.Generator().manual_seed(10 * k + i)) * 1e-3)
        scale.fill_(0.3 + 0.1 * k)
        other, copies = twin_of(opt, params, bits, 1)             # (the recorded step is the second)
        other.step(grad_scale=scale.clone())
        if k % 2:
            torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        same(opt, params, other, copies)
        # eager steps with other gradients, and from k = 2 on with fewer of them: tables of their own
        for p, g in zip(params, recorded):
            p.grad = torch.full_like(g, 1e-3)
        if k >= 2:
            params[1].grad = None
        opt.step()
        torch.cuda.synchronize()
        for p, g in zip(params, recorded):
            p.grad = g


@pytest.mark.parametrize("bits", [32, 8])
def test_tables_of_a_graph_outlive_the_optimizer(bits):
    from muon_amd import engine
    params = make([3000], F32)
    opt = optimizer(params, bits)
    opt.step()
    before = len(engine._TABLES_OF_GRAPHS)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        opt.step()
        opt.step()                                # the same tables: kept once
    assert len(engine._TABLES_OF_GRAPHS) == before + 1
    other, copies = twin_of(opt, params, bits, 1)
    for _ in range(2):
        other.step()
    states = {p: dict(s) for p, s in opt.state.items()}
    del opt
    fill = [torch.full((3000,), 255, dtype=torch.uint8, device=DEV) for _ in range(64)]      # takes memory that was given back
    graph.replay()
    torch.cuda.synchronize()
    assert len(fill) == 64 and torch.equal(params[0], copies[0])
    assert all(torch.equal(v, other.state[copies[0]][k]) for k, v in states[params[0]].items() if isinstance(v, torch.Tensor))


def test_a_step_with_a_graph_of_its_own_is_not_captured():
    params = make([100], F32)
    opt = optimizer(params, 32, use_graph=True)
    opt.step()
    other = make([100], F32)
    plain = optimizer(other, 32)
    plain.step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        plain.step()
        with pytest.raises(muon_amd.MuonAmdError, match="captured"):
            opt.step()
    assert opt.state[params[0]]["step"] == 1
