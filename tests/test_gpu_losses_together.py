"""The losses and the balanced router as a training step uses them together, and in the example.

Bounds.  u = 2^-8 (bf16).  The gradients are held against those of the same model in 64 bits from the same bf16 values: every
tensor that is rounded on the way (hidden states of the head, their gradient, the router's logits' gradient) is off by u of itself, and each gradient here passes at
most four such roundings: 8 u of its norm.  The loss passes none but the hidden states' own: 4 u of itself."""
import importlib.util
import os

import pytest
import torch

import muon_amd

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
u = 2.0 ** -8
T, D, V, E, K, G = 600, 128, 1000, 32, 4, 8


def leaves():
    g = torch.Generator().manual_seed(0)
    make = lambda *s, std: (torch.randn(*s, generator=g) * std).bfloat16()
    x, router, head = make(T, D, std=1.0), make(D, E, std=D ** -0.5 * 1.5), make(V, D, std=2 * D ** -0.5)
    target = torch.randint(V, (T,), generator=g)
    target[torch.rand(T, generator=g) < 0.2] = -100
    values, index = (torch.randn(T, 5, generator=g) * 2 + 4).bfloat16(), torch.argsort(torch.rand(T, V, generator=g), 1)[:, :5]
    index[::7] = -1
    bias = torch.randn(E, generator=g) * 0.05
    experts = make(E, D, std=1.0)
    return x, router, head, experts, target, values, index, bias


def step(x, router, head, experts, target, values, index, bias):
    """A token gets its experts' vectors by the weights it gives them; head, z-loss, teacher and router's losses on top."""
    r = muon_amd.route_topk(x @ router, K, scores="sigmoid", bias=bias, groups=G, groups_kept=3)
    share = torch.zeros(T, E, device=DEV).scatter(1, r.indices.long(), r.weights)
    y = (x.float() + share @ experts.float()).bfloat16()
    out = muon_amd.linear_cross_entropy(y, head, target)
    taught = muon_amd.distill_topk(y @ head.t(), values, index, temperature=2.0)
    return out.loss + 1e-3 * out.lse.square().mean() + 0.5 * taught + 0.01 * r.balance_loss + 1e-3 * r.z_loss, r.indices


def exact(x, router, head, experts, target, values, index, bias, chosen):
    x, router, head, experts = (t.detach().double().requires_grad_() for t in (x, router, head, experts))
    logits = (x @ router)
    s = torch.sigmoid(logits)
    w = s.gather(1, chosen)
    w = w / w.sum(1, keepdim=True)
    y = x + (w[..., None] * experts[chosen]).sum(1)
    lx = y @ head.t()
    on = target != -100
    lse = torch.logsumexp(lx, 1)
    ce = torch.nn.functional.cross_entropy(lx, target)
    there = index >= 0
    some = there.any(1)
    t = torch.where(there, values.double() / 2, -torch.inf)[some]
    q, lq = torch.softmax(t, 1), torch.log_softmax(t, 1)
    lp = torch.log_softmax(lx[some] / 2, 1).gather(1, index[some])
    taught = 4 * torch.where(q > 0, q * (lq - lp), 0.0).sum(1).mean()
    counts = torch.bincount(chosen.flatten(), minlength=E).double()
    balance = E * (counts / (T * K) * (s / s.sum(1, keepdim=True)).mean(0)).sum()
    z = torch.logsumexp(logits, 1).square().mean()
    total = ce + 1e-3 * torch.where(on, lse, 0.0).square().sum() / T + 0.5 * taught + 0.01 * balance + 1e-3 * z
    return total, torch.autograd.grad(total, (x, router, head, experts))


def test_a_step_with_all_of_them():
    args = [t.to(DEV) for t in leaves()]
    for t in args[:4]:
        t.requires_grad_()
    total, chosen = step(*args)
    grads = torch.autograd.grad(total, args[:4])
    want, wgrads = exact(*args[:4], *(t.cpu().to(DEV) for t in args[4:]), chosen.long())
    assert abs(float(total.detach()) - float(want.detach())) <= 4 * u * float(want.detach())
    for g, w in zip(grads, wgrads):
        assert (g.double() - w).norm() <= 8 * u * w.norm()


def test_a_captured_step():
    args = [t.to(DEV) for t in leaves()]
    for t in args[:4]:
        t.requires_grad_()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.autograd.grad(step(*args)[0], args[:4])
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        total, _ = step(*args)
        grads = torch.autograd.grad(total, args[:4])
    for round in range(3):
        with torch.no_grad():
            args[0].mul_(0.5 + 0.5 * round)
            args[4].copy_(args[4].roll(1))
        graph.replay()
        torch.cuda.synchronize()
        again, _ = step(*args)
        assert torch.equal(again.detach(), total.detach())
        for a, b in zip(grads, torch.autograd.grad(again, args[:4])):
            assert torch.equal(a, b)


def test_a_capture_while_an_eager_graph_holds_a_leaf_is_refused():
    """Recorded, its backward pass would end the process: each operator says so in the forward pass, for a leaf and for what follows from one."""
    g = torch.Generator().manual_seed(0)
    x, w = (torch.randn(8, 64, generator=g).bfloat16().to(DEV).requires_grad_() for _ in range(2))
    t, i = torch.arange(8, device=DEV), torch.zeros(8, 2, dtype=torch.int32, device=DEV)
    v, ones = torch.zeros(8, 2, device=DEV), torch.ones(64, device=DEV, requires_grad=True)
    calls = (lambda x: muon_amd.linear_cross_entropy(x, w, t).loss, lambda x: muon_amd.distill_topk(x, v, i),
             lambda x: muon_amd.route_topk(x, 2).balance_loss, lambda x: muon_amd.route_topk(x, 2, scores="sigmoid").balance_loss,
             lambda x: muon_amd.residual_norm(x, x, ones, ones)[0])
    for call in calls:
        for of in (lambda: x, lambda: x * 2):
            kept = call(of())
            graph = torch.cuda.CUDAGraph()
            with pytest.raises(muon_amd.MuonAmdError, match="default stream"):
                with torch.cuda.graph(graph):
                    call(of())
            with torch.cuda.graph(torch.cuda.CUDAGraph()):       # without a gradient there is nothing to refuse
                with torch.no_grad():
                    call(of())
            del kept


def example():
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "train_moe.py")
    spec = importlib.util.spec_from_file_location("train_moe", path)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


def test_the_example_with_each_option():
    e = example()
    for options in (dict(fused_head=True), dict(distill=0.5), dict(balanced=True), dict(fused_head=True, distill=0.3, balanced=True, state_bits=32)):
        losses = e.train(steps=4, width=96, layers=2, experts=4, **options)
        assert len(losses) == 4 and all(0 < l < 20 for l in losses)
    # the first loss is that of the default, to the rounding of its logits
    assert abs(e.train(steps=1, width=96, layers=2, experts=4, fused_head=True)[0] - e.train(steps=1, width=96, layers=2, experts=4)[0]) <= 4 * u * 5


def test_the_example_head_has_the_gradients_of_torch():
    e = example()
    torch.manual_seed(0)
    model = e.Model(96, 1, 4, 2).to(DEV)
    ids = next(e.batches(torch.device(DEV)))
    with torch.no_grad():
        model.head.normal_(0, 0.2)
    y, _, _ = model(ids[:, :-1])
    a = muon_amd.linear_cross_entropy(y, model.head.t().bfloat16(), ids[:, 1:]).loss
    b = torch.nn.functional.cross_entropy(model.logits(y).flatten(0, 1), ids[:, 1:].flatten())
    assert abs(float(a.detach()) - float(b.detach())) <= 4 * u * float(b.detach())
    got = torch.autograd.grad(a, (model.head, model.embedding), retain_graph=True)
    want = torch.autograd.grad(b, (model.head, model.embedding))
    for g, w in zip(got, want):
        assert (g - w).norm() <= 8 * u * w.norm()
