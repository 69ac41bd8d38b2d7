"""AdamW over lists of tensors that change between steps: converted, resized and replaced parameters, other subsets with a
gradient.  Each step is held to the formulas in 64 bits (the bounds of test_gpu_adamw), or to a fresh optimizer's bits."""
import pytest
import torch

import muon_amd
from test_gpu_adamw import BETAS, EPS, LR, WD, make, step_and_check

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
F32, BF16 = torch.float32, torch.bfloat16


def optimizer(params, bits, **options):
    return muon_amd.AdamW(params, lr=LR, betas=BETAS, eps=EPS, weight_decay=WD, state_bits=bits, **options)


def twin_of(opt, params, bits):
    """An optimizer of its own over copies of the parameters, gradients and states as they are."""
    copies = [torch.nn.Parameter(p.detach().clone()) for p in params]
    for q, p in zip(copies, params):
        q.grad = p.grad.clone()
    other = optimizer(copies, bits)
    for q, p in zip(copies, params):
        if len(opt.state[p]):
            other.state[q].update({k: v.clone() if isinstance(v, torch.Tensor) else v for k, v in opt.state[p].items()})
    return other, copies


def same_as_a_fresh_one(opt, params, bits):
    other, copies = twin_of(opt, params, bits)
    opt.step()
    other.step()
    for p, q in zip(params, copies):
        assert torch.equal(p, q)
        for k, v in opt.state[p].items():
            assert torch.equal(v, other.state[q][k]) if isinstance(v, torch.Tensor) else v == other.state[q][k]


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("first,then", [(F32, BF16), (BF16, F32)], ids=["to-bf16", "to-fp32"])
def test_parameters_converted_between_steps(first, then, bits):
    params = make([5000, (129, 65), 8193], first)
    opt = optimizer(params, bits)
    for _ in range(2):
        step_and_check(opt, params, bits)
    for p in params:                              # what Module.bfloat16() and .float() do
        grad = p.grad
        p.grad = None
        p.data = p.data.to(then)
        p.grad = grad.to(then)
    for _ in range(3):
        same_as_a_fresh_one(opt, params, bits)
    step_and_check(opt, params, bits)


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("sizes", [(20000, 300), (300, 20000)], ids=["smaller", "larger"])
def test_parameters_resized_and_replaced(sizes, bits):
    before, after = sizes
    params = make([before, 70], F32)
    opt = optimizer(params, bits)
    for _ in range(2):
        opt.step()
    resized, other = make([after, 70], F32, seed=1)
    p = params[0]
    p.grad = None
    p.data = resized.data
    p.grad = resized.grad
    opt.state.pop(p)                              # its state starts anew, its neighbour's goes on: two launches
    for _ in range(3):
        step_and_check(opt, params, bits)
    opt.state.pop(params[1])
    params[1] = opt.param_groups[0]["params"][1] = make([before], F32, seed=2)[0]
    for _ in range(3):
        step_and_check(opt, params, bits)


@pytest.mark.parametrize("bits", [32, 8])
def test_other_parameters_have_gradients(bits):
    params = make([1000, 1000, 8192, 40], F32)
    grads = [p.grad for p in params]
    opt = optimizer(params, bits)
    for kept in ((0, 1, 2, 3), (1, 3), (0, 2), (0, 1, 2, 3), (2,), (1, 3), (0, 1, 2, 3)):
        for i, p in enumerate(params):
            p.grad = grads[i] if i in kept else None
        untouched = [p.detach().clone() for p in params]
        step_and_check(opt, [params[i] for i in kept], bits)
        assert all(torch.equal(p, q) for i, (p, q) in enumerate(zip(params, untouched)) if i not in kept)
    assert len(opt._adamw_engines) <= 4           # launches of one step, however many lists there were


@pytest.mark.parametrize("bits", [32, 8])
def test_recorded_steps_follow_a_conversion(bits):
    pairs = [make([1000, (129, 65)], F32) for _ in range(2)]
    opts = [optimizer(ps, bits, use_graph=g) for ps, g in zip(pairs, (False, True))]
    for k in range(6):
        for opt, ps in zip(opts, pairs):
            if k == 3:
                for p in ps:
                    grad = p.grad
                    p.grad = None
                    p.data = p.data.bfloat16()
                    p.grad = grad.bfloat16()
            opt.step()
        torch.cuda.synchronize()
        for p, q in zip(*pairs):
            # (the bias corrections are formed on the device in a recorded step: a rounding each; in bf16 one of its steps)
            torch.testing.assert_close(p.float(), q.float(), rtol=2.0 ** -7 if k >= 3 else 1e-5, atol=0 if k >= 3 else 1e-7)


def test_lists_that_change_on_other_streams():
    params = make([5000, 3000], F32)
    grads = [p.grad for p in params]
    opt = optimizer(params, 8)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for k in range(6):
        params[1].grad = grads[1] if k % 3 else None
        s = streams[k % 2]
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            step_and_check(opt, params if k % 3 else params[:1], 8)
        torch.cuda.current_stream().wait_stream(s)
