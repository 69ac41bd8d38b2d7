"""residual_norm and route_topk, forward and backward, recorded into a HIP graph: every replay is the eager result, with the
program's own work between replays."""
import pytest
import torch

import muon_amd

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def both(t):
    h, y = muon_amd.residual_norm(t["x"], t["block"], t["post"], t["pre"], gate=t["gate"], scale=t["scale"])
    r = muon_amd.route_topk(t["logits"], 3, mask=t["mask"])
    leaves = [t[n] for n in ("x", "block", "post", "pre", "gate", "scale", "logits")]
    grads = torch.autograd.grad((h, y, r.weights, r.balance_loss, r.z_loss), leaves, (t["dh"], t["dy"], t["dw"], t["one"], t["one"]))
    return [h, y, *r, *grads]


def fill(t, seed):
    g = torch.Generator().manual_seed(seed)
    for n, v in t.items():
        new = torch.rand(v.shape, generator=g) < 0.8 if v.dtype == torch.bool else torch.randn(v.shape, generator=g)
        v.data.copy_(new)


def test_replays():
    bf, f = torch.bfloat16, torch.float32
    shapes = dict(x=((700, 520), f), block=((700, 520), bf), post=((520,), f), pre=((520,), f), gate=((700, 520), bf), scale=((1,), f),
                  logits=((900, 70), bf), mask=((900,), torch.bool), dh=((700, 520), f), dy=((700, 520), bf), dw=((900, 3), f), one=((), f))
    t = {n: torch.zeros(s, dtype=d, device=DEV) for n, (s, d) in shapes.items()}
    for n in ("x", "block", "post", "pre", "gate", "scale", "logits"):
        t[n].requires_grad_()
    fill(t, 0)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            both(t)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        recorded = both(t)
    for k in range(5):
        fill(t, k + 1)
        want = [v.detach().clone() for v in both(t)]
        torch.cuda.synchronize()
        graph.replay()
        if k % 2:
            torch.cuda.synchronize()
        for a, b in zip(recorded, want):
            assert torch.equal(a, b)
