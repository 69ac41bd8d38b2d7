"""A forward pass captured while an eager graph of the same leaves lives: what the refusal advises works, and gives what the eager call gives (GPU)."""
import pytest
import torch

import muon_amd

DEV = "cuda:0"


@pytest.mark.gpu
@pytest.mark.parametrize("name", ["head", "distill", "route", "scored", "norm"])
def test_the_two_ways_out(name):
    g = torch.Generator().manual_seed(0)
    x, w = (torch.randn(8, 64, generator=g).bfloat16().to(DEV).requires_grad_() for _ in range(2))
    t, i = torch.arange(8, device=DEV), torch.zeros(8, 2, dtype=torch.int32, device=DEV)
    v, ones = torch.zeros(8, 2, device=DEV), torch.ones(64, device=DEV, requires_grad=True)
    call = {"head": lambda: muon_amd.linear_cross_entropy(x, w, t).loss, "distill": lambda: muon_amd.distill_topk(x, v, i),
            "route": lambda: muon_amd.route_topk(x, 2).weights, "scored": lambda: muon_amd.route_topk(x, 2, scores="sigmoid").weights,
            "norm": lambda: muon_amd.residual_norm(x, x, ones, ones)[0]}[name]
    kept = call()
    with pytest.raises(muon_amd.MuonAmdError, match="release it.*torch.no_grad"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            call()

    def replays(graph, out):
        for step in range(3):
            with torch.no_grad():
                x.mul_(0.5 + step)
                want = call()
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, want)

    graph = torch.cuda.CUDAGraph()
    with torch.no_grad(), torch.cuda.graph(graph):
        out = call()
    replays(graph, out)
    del kept, out
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()                                             # (nothing holds the leaves now)
    replays(graph, out.detach())
