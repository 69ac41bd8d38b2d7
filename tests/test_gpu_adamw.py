"""AdamW over many tensors, states in 32 and in 8 bits, against the formulas in 64 bits (GPU), its refusals, and the
ways a program keeps it: state dicts, copies, graphs, the auxiliary groups of the Muon classes.

Bounds.  u = 2^-24 (fp32) and 2^-8 (bf16) are unit roundoffs.  A moment is a lerp of two roundings and one of its operands:
4 u (|old| + |new|) bounds it.  The parameter takes p (1 - lr wd) - a m / d: two roundings at p, and at the update the
error of m, a square root, a division and two products, together below 16 u (|old| + |new|) a / d with a, d exact; then one
rounding to its type.  What 8 bits hold goes by the moment in fp32 (a bf16 gradient times 0.1 can lie on the boundary between two shared
exponents in 64 bits, and the square of a tiny gradient is zero in fp32): product, difference, and one fused product and
sum.  A code is floor(y) for y = |x| / step + dither, floor(y - 2^-16) or floor(y + 2^-16)."""
import copy
import math

import numpy as np
import pytest
import torch

import muon_amd

gpu = pytest.mark.gpu
DEV = "cuda:0"
U32, U16 = 2.0 ** -24, 2.0 ** -8
LR, BETAS, EPS, WD = 3e-3, (0.9, 0.95), 1e-8, 0.01
SHARED = 128
FORMATS = {"m": dict(top=15, carry=14 / 16, factor=0xC13FA9), "v": dict(top=31, carry=15 / 16, factor=0x91E10D)}


# ---- the 8-bit format in 64 bits ----------------------------------------------------------------------------
def blocks_of(x):
    return np.concatenate([x, np.zeros(-len(x) % SHARED)]).reshape(-1, SHARED)


def shared_exponent(x, kind):
    """E of every block of a moment."""
    mantissa, e = np.frexp(np.abs(blocks_of(x)).max(1))           # mantissa in [1/2, 1)
    return np.where(mantissa == 0, 0, np.where(mantissa > FORMATS[kind]["carry"], e, e - 1) + 127)


def mix(t):
    for factor, shift in ((0x9E3779B9, 16), (0xC13FA9A9, 15), (0x91E10DA5, 16)):
        t = t * factor & 0xFFFFFFFF
        t ^= t >> shift
    return t


def rounded(x, kind, step, slack, E, first=0):
    """The value that x's code stands for, with y = |x| / step + dither moved by `slack`; first: the place of x[0]."""
    f = FORMATS[kind]
    b, E = blocks_of(x), E[:, None]
    power = np.maximum(np.frexp(np.abs(b))[1] - 1, E - 127 - (f["top"] - 1))
    i = (np.arange(b.size, dtype=np.uint64) + np.uint64(first)).reshape(b.shape) % np.uint64(1 << 32)
    h = (i * np.uint64(0x9E3779B9) + np.uint64(mix(step))) % np.uint64(1 << 32)
    u = ((h ^ h >> np.uint64(15)) % np.uint64(1 << 24) * np.uint64(f["factor"]) % np.uint64(1 << 32) >> np.uint64(12)).astype(np.float64) / (1 << 20)
    y = np.ldexp(np.abs(b), 3 - power) + u + slack
    q = np.floor(np.maximum(y, 0))
    if kind == "v":
        q = np.where(b > 0, np.maximum(q, 1), 0)
    return (np.sign(b) * np.ldexp(q, power - 3) * (np.abs(b).max(1, keepdims=True) > 0)).reshape(-1)[:len(x)]


def values(code, E, kind):
    code, E = code.astype(np.int64).ravel(), np.repeat(E.astype(np.int64), SHARED)[:code.size]
    low = code & (0x7F if kind == "m" else 0xFF)
    e, f = low >> 3, low & 7
    x = np.where(e > 0, np.ldexp(1 + f / 8, e - FORMATS[kind]["top"]), np.ldexp(f / 8, 1 - FORMATS[kind]["top"])) * np.ldexp(1.0, E - 127)
    x = np.where((kind == "m") & (code > 0x7F), -x, x)
    return np.where(E == 255, np.nan, np.where(E == 0, 0.0, x))


# ---- one step against 64 bits ------------------------------------------------------------------------------------
def moments_of(opt, p, bits):
    s = opt.state[p]
    if bits == 32:
        return [s[k].cpu().double().numpy().ravel() for k in ("exp_avg", "exp_avg_sq")]
    return [values(s[k].cpu().numpy(), s[k + "_exponent"].cpu().numpy(), kind) for k, kind in (("exp_avg", "m"), ("exp_avg_sq", "v"))]


def lerp32(old, new, w):
    """old + w (new - old) in the roundings of fp32 (w below one half, else from the other end)."""
    d = (new - old).astype(np.float32).astype(np.float64)
    return (old + w * d if w < 0.5 else new - d * np.float64(np.float32(1) - np.float32(w))).astype(np.float32).astype(np.float64)


def step_and_check(opt, params, bits, scale=None, lr=LR, wd=WD, betas=BETAS, eps=EPS, check_param=True):
    before = []
    for p in params:
        has = len(opt.state[p]) > 0
        m, v = moments_of(opt, p, bits) if has else (np.zeros(p.numel()), np.zeros(p.numel()))
        before.append((p.detach().cpu().double().numpy().ravel(), m, v, opt.state[p]["step"] if has else 0))
    opt.step(**({} if scale is None else {"grad_scale": torch.tensor(scale, device=DEV)}))
    torch.cuda.synchronize()
    for p, (p0, m0, v0, t0) in zip(params, before):
        t = t0 + 1
        assert opt.state[p]["step"] == t
        c = np.float64(np.float32(1.0 if scale is None else scale))
        g = p.grad.cpu().double().numpy().ravel() * c
        w1, w2 = np.float64(np.float32(1 - betas[0])), np.float64(np.float32(1 - betas[1]))
        m, v = m0 + w1 * (g - m0), v0 + w2 * (g * g - v0)
        m1, v1 = moments_of(opt, p, bits)
        if bits == 32:
            np.testing.assert_array_less(np.abs(m1 - m), 4 * U32 * (np.abs(m0) + np.abs(g)) + 1e-44)
            np.testing.assert_array_less(np.abs(v1 - v), 4 * U32 * (np.abs(v0) + g * g) + 1e-44)
        else:
            g32 = g.astype(np.float32).astype(np.float64)
            for got, want, in32, kind in ((m1, m, lerp32(m0, g32, w1), "m"),
                                          (v1, v, lerp32(v0, (g32 * g32).astype(np.float32).astype(np.float64), w2), "v")):
                key = "exp_avg" if kind == "m" else "exp_avg_sq"
                E = shared_exponent(in32, kind)
                np.testing.assert_array_equal(opt.state[p][key + "_exponent"].cpu().numpy(), E)
                lo, hi = (np.abs(rounded(in32, kind, t, slack, E)) for slack in (-2.0 ** -16, 2.0 ** -16))
                assert ((np.abs(got) >= lo) & (np.abs(got) <= hi)).all()
                assert ((np.sign(got) == np.sign(in32)) | (got == 0)).all()
                np.testing.assert_array_less(np.abs(in32 - want), 4 * U32 * (np.abs(m0) + np.abs(g)) + 1e-44
                                             if kind == "m" else 4 * U32 * (np.abs(v0) + g * g) + 1e-44)
        if check_param:
            a = lr / (1 - betas[0] ** t)
            d = np.sqrt(v / (1 - betas[1] ** t)) + eps
            want = p0 * (1 - lr * wd) - a * m / d
            got = p.detach().cpu().double().numpy().ravel()
            u = U32 if p.dtype == torch.float32 else U16
            np.testing.assert_array_less(np.abs(got - want), u * np.abs(want) + 2 * U32 * np.abs(p0) +
                                         16 * U32 * a * (np.abs(m0) + np.abs(g)) / d + 1e-38)


def make(sizes, dtype, seed=0, offset=0, gstd=1e-3):
    """Parameters and gradients as views into flat buffers, `offset` elements off the buffer's start."""
    gen = torch.Generator().manual_seed(seed)
    params = []
    for n in sizes:
        shape = n if isinstance(n, tuple) else (n,)
        numel = math.prod(shape)
        buf = torch.randn(2, numel + 16, generator=gen) * torch.tensor([[0.05], [gstd]])
        buf = buf.to(dtype).to(DEV)
        p = torch.nn.Parameter(buf[0, offset:offset + numel].view(shape))
        p.grad = buf[1, offset + 3:offset + 3 + numel].view(shape)
        params.append(p)
    return params


SIZES = [[1], [7, 8, 9], [127, 128, 129, 255], [4095, 4096, 4097], [(3, 5), 0, 8191, (8, 1024), 8193], [(129, 257), 16384 + 5]]


@gpu
@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("offset", [0, 1, 5])
@pytest.mark.parametrize("sizes", SIZES, ids=str)
def test_steps(sizes, offset, dtype, bits):
    params = make(sizes, dtype, seed=offset, offset=offset)
    opt = muon_amd.AdamW(params, lr=LR, betas=BETAS, eps=EPS, weight_decay=WD, state_bits=bits)
    for k in range(3):
        step_and_check(opt, [p for p in params if p.numel()], bits, scale=None if k != 1 else 0.37)


@gpu
@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("betas", [(0.0, 0.0), (0.3, 0.5), (0.95, 0.999)])
def test_other_betas(betas, bits):
    params = make([1000, 300], torch.float32)
    opt = muon_amd.AdamW(params, lr=LR, betas=betas, eps=EPS, weight_decay=WD, state_bits=bits)
    for k in range(3):
        step_and_check(opt, params, bits, betas=betas)


@gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_types_mixed_in_one_launch(bits):
    params = [p for ps in (make([300, 9000], torch.bfloat16), make([8193, 40], torch.float32)) for p in ps]
    opt = muon_amd.AdamW(params, lr=LR, betas=BETAS, eps=EPS, weight_decay=WD, state_bits=bits)
    for k in range(2):
        step_and_check(opt, params, bits)


@gpu
def test_gradients_over_many_powers_and_zeros():
    # from 2^-60 to 2^40 within one block of 128, blocks of zeros, and a block whose largest is far below the others
    params = make([128 * 6 + 50], torch.float32)
    g = params[0].grad
    g.mul_(torch.exp2(torch.linspace(-50, 50, 128, device=DEV).repeat(7)[:g.numel()]))
    g[256:384] = 0
    g[384:512] *= 1e-30
    opt = muon_amd.AdamW(params, lr=LR, betas=BETAS, eps=EPS, weight_decay=WD, state_bits=8)
    step_and_check(opt, params, 8)
    step_and_check(opt, params, 8)
    m, v = opt.state_values()[0]
    assert (m[256:384] == 0).all() and (v[256:384] == 0).all()
    # (the codes: bf16 does not hold the values of a block whose largest is 1e-38)
    assert ((opt.state[params[0]]["exp_avg_sq"] > 0) | (0.05 * g.square() < 2.0 ** -148)).all(), "v above zero does not become zero"


@gpu
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf"), 1e30])
def test_what_is_not_finite_shows(bad):
    params = make([1000], torch.float32)
    opts = [muon_amd.AdamW(make([1000], torch.float32), lr=LR, state_bits=b) for b in (8, 32)]
    for opt in opts:
        p = opt.param_groups[0]["params"][0]
        p.grad[300] = bad                       # in the block 256 .. 383 (1e30: its square overflows)
        opt.step()
        p.grad.copy_(params[0].grad)
        opt.step()
        poisoned = ~torch.isfinite(p.detach())
        where = torch.arange(1000, device=DEV)
        if bad != 1e30:
            assert poisoned[300]
        if opt._state_bits == 8:
            inside = (where >= 256) & (where < 384)
            assert torch.equal(poisoned, inside)
            m, v = opt.state_values()[0]
            assert torch.equal(torch.isnan(m), inside) and torch.equal(torch.isnan(v), inside)
        else:
            assert not poisoned[where != 300].any()


@gpu
def test_state_values_are_what_the_codes_stand_for():
    params = make([1, 130, (65, 127)], torch.bfloat16)
    opt = muon_amd.AdamW(params, state_bits=8)
    opt.step()
    outs = [tuple(torch.full((p.numel() + 1,), 7.0, dtype=torch.bfloat16, device=DEV)[1:] for _ in range(2)) for p in params]
    got = opt.state_values(out=outs)
    as_lists = opt.state_values(out=[[torch.empty_like(t) for t in pair] for pair in outs])       # (the general way)
    assert all(torch.equal(a, b) for x, y in zip(got, as_lists) for a, b in zip(x, y))
    for p, (m, v), fresh in zip(params, got, opt.state_values()):
        for t, k, kind, f in ((m, "exp_avg", "m", fresh[0]), (v, "exp_avg_sq", "v", fresh[1])):
            want = values(opt.state[p][k].cpu().numpy(), opt.state[p][k + "_exponent"].cpu().numpy(), kind)
            np.testing.assert_array_equal(t.cpu().double().numpy().ravel(), want)
            assert torch.equal(f.ravel(), t.ravel()) and f.shape == p.shape
    # the first moment's codes are float8_e4m3fn's
    p = params[2]
    e4m3 = opt.state[p]["exp_avg"].view(torch.float8_e4m3fn).float().cpu().double().numpy().ravel()
    E = np.repeat(opt.state[p]["exp_avg_exponent"].cpu().numpy().astype(np.int64), SHARED)[:p.numel()]
    np.testing.assert_array_equal(np.ldexp(e4m3, E - 135), values(opt.state[p]["exp_avg"].cpu().numpy(), opt.state[p]["exp_avg_exponent"].cpu().numpy(), "m"))


@gpu
def test_moments_follow_slow_averages():
    """beta2 = 0.999 moves v by at most a thousandth of itself, far below a code's step: the dither carries it."""
    n, steps = 4096, 600
    p = torch.nn.Parameter(torch.zeros(n, device=DEV))
    p.grad = torch.exp(0.7 * torch.randn(n, generator=torch.Generator().manual_seed(1))).to(DEV)
    opt = muon_amd.AdamW([p], lr=0.0, betas=(0.99, 0.999), state_bits=8)
    g = p.grad.clone()
    for k in range(steps):
        if k == steps // 2:
            p.grad.mul_(0.5)                   # the averages have to come down again
        opt.step()
    m, v = (t.double() for t in opt.state_values()[0])
    half = steps // 2
    wm = (1 - 0.99 ** half) * 0.99 ** half + 0.5 * (1 - 0.99 ** half)
    wv = (1 - 0.999 ** half) * 0.999 ** half + 0.25 * (1 - 0.999 ** half)
    # a code alone is up to 1/8 off; the mean over 4096 elements of a rounding that is right on average is far nearer
    assert abs(float((m / g.double()).mean()) / wm - 1) < 0.01
    assert abs(float((v / g.double().square()).mean()) / wv - 1) < 0.01


@gpu
def test_strided_tensors_missing_gradients_and_groups():
    base = torch.randn(40, 30, device=DEV)
    a = torch.nn.Parameter(base.t())                              # not row-major
    b, c = (torch.nn.Parameter(torch.randn(77, device=DEV)) for _ in range(2))
    a.grad = torch.randn(60, 40, device=DEV)[::2]
    b.grad = torch.randn(154, device=DEV)[::2]
    opt = muon_amd.AdamW([dict(params=[a, c], lr=LR), dict(params=[b], lr=LR, weight_decay=WD)], betas=BETAS, eps=EPS, weight_decay=WD, state_bits=8)
    before = c.detach().clone()
    step_and_check(opt, [a, b], 8)
    assert torch.equal(c, before) and len(opt.state[c]) == 0      # no gradient: left alone
    c.grad = torch.randn(77, device=DEV)
    step_and_check(opt, [a, b, c], 8)                             # two step counts in one group
    assert opt.state[c]["step"] == 1 and opt.state[a]["step"] == 2


@gpu
@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("how", ["state_dict", "deepcopy"])
def test_state_survives(bits, how):
    params = make([1000, (33, 65)], torch.bfloat16)
    opt = muon_amd.AdamW(params, lr=LR, state_bits=bits)
    for _ in range(2):
        opt.step()
    if how == "deepcopy":
        other = copy.deepcopy(opt)
        twins = other.param_groups[0]["params"]
        for q, p in zip(twins, params):
            q.grad = p.grad.clone()
    else:
        twins = [torch.nn.Parameter(p.detach().clone()) for p in params]
        for q, p in zip(twins, params):
            q.grad = p.grad.clone()
        other = muon_amd.AdamW(twins, lr=LR, state_bits=bits)
        other.load_state_dict(copy.deepcopy(opt.state_dict()))
    opt.step()
    other.step()
    for p, q in zip(params, twins):
        assert torch.equal(p, q)
        for k in opt.state[p]:
            x, y = opt.state[p][k], other.state[q][k]
            assert x.dtype == y.dtype and torch.equal(x, y) if isinstance(x, torch.Tensor) else x == y


@gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_recorded_steps_are_the_eager_ones(bits):
    pairs = [make([1000, (129, 65)], torch.bfloat16) for _ in range(2)]
    opts = [muon_amd.AdamW(ps, lr=LR, state_bits=bits, use_graph=g) for ps, g in zip(pairs, (False, True))]
    scale, graphs, kept = torch.ones((), device=DEV), set(), []
    for k in range(5):
        scale.fill_(0.5 + 0.1 * k)
        for opt, ps in zip(opts, pairs):
            for group in opt.param_groups:
                group["lr"] = LR / (k + 1)
            kept.append(scale.clone())                            # (a tensor of its own at every step)
            opt.step(grad_scale=kept[-1])
            graphs.add(id(opts[1]._graphs[torch.device(DEV)].graph) if opt is opts[1] else None)
            if k % 2:
                for p in ps:
                    p.grad.mul_(0.75)
            if k == 3:
                for p in ps:
                    p.grad = p.grad.clone()                       # the gradients move
        torch.cuda.synchronize()
        for p, q in zip(*pairs):
            # (the bias corrections are formed on the device in a recorded step)
            torch.testing.assert_close(p.float(), q.float(), rtol=2 * U16, atol=0)
            assert opts[0].state[p]["step"] == opts[1].state[q]["step"]
    assert opts[1]._graphs[torch.device(DEV)].replays == 5 and len(graphs) == 2      # recorded once (and None)


@gpu
def test_auxiliary_groups_of_the_muon_classes():
    def build(bits):
        gen = torch.Generator().manual_seed(3)
        w = torch.nn.Parameter((torch.randn(64, 128, generator=gen) * 0.05).to(DEV))
        aux = [torch.nn.Parameter((torch.randn(*s, generator=gen) * 0.05).to(DEV)) for s in ((300, 64), (64,))]
        for p in (w, *aux):
            p.grad = (torch.randn(p.shape, generator=gen) * 1e-3).to(DEV)
        opt = muon_amd.MuonWithAuxAdam([dict(params=[w], use_muon=True, lr=0.02), dict(params=aux, use_muon=False, lr=LR, betas=BETAS, eps=EPS, weight_decay=WD)],
                                       adam_state_bits=bits)
        return opt, w, aux

    plain, w0, aux0 = build(None)
    plain.step()
    for bits in (32, 8):
        opt, w, aux = build(bits)
        step_and_check_aux = [p.detach().clone() for p in aux]
        step_and_check(opt, aux, bits, check_param=True)
        assert torch.equal(w, w0) and not any(torch.equal(p, q) for p, q in zip(aux, step_and_check_aux))
        for p, q in zip(aux, aux0):
            torch.testing.assert_close(p, q, rtol=1e-5, atol=1e-8)
        again = copy.deepcopy(opt)
        assert again._adam_state_bits == bits
        again.step()
        fresh, _, _ = build(bits)
        fresh.load_state_dict(opt.state_dict())
        assert fresh.state[fresh.param_groups[1]["params"][0]]["exp_avg"].dtype == (torch.float32 if bits == 32 else torch.uint8)


@gpu
def test_other_stream():
    params = make([100000], torch.float32)
    opt = muon_amd.AdamW(params, lr=LR, betas=BETAS, eps=EPS, weight_decay=WD, state_bits=8)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step_and_check(opt, params, 8)
        step_and_check(opt, params, 8)


@gpu
def test_refusals_on_the_device():
    p = torch.nn.Parameter(torch.zeros(10, device=DEV))
    p.grad = torch.zeros(10, device=DEV)
    opt = muon_amd.AdamW([p], state_bits=8)
    with pytest.raises(TypeError):
        opt.step(grad_scale=torch.ones(2, device=DEV))
    with pytest.raises(TypeError):
        opt.step(grad_scale=torch.ones((), device=DEV, dtype=torch.float64))
    with pytest.raises(muon_amd.MuonAmdError):
        opt.step(grad_scale=torch.ones(()))
    opt.step()
    with pytest.raises(ValueError):
        opt.state_values(out=[])
    with pytest.raises(ValueError):
        opt.state_values(out=[(torch.zeros(10, device=DEV), torch.zeros(10, device=DEV))])
    opt.state[p]["exp_avg"] = torch.zeros(10, device=DEV)         # a state of another kind
    with pytest.raises(NotImplementedError):
        opt.step()
    assert opt.state[p]["step"] == 1
    half = torch.nn.Parameter(torch.zeros(10, device=DEV, dtype=torch.float16))
    half.grad = torch.zeros_like(half)
    with pytest.raises(NotImplementedError):
        muon_amd.AdamW([half]).step()


def test_refusals():
    p = torch.nn.Parameter(torch.zeros(10))
    p.grad = torch.zeros(10)
    for bad in (dict(state_bits=16), dict(betas=(1.0, 0.9)), dict(betas=(0.9, -0.1)), dict(lr=-1.0), dict(eps=-1e-8), dict(weight_decay=-1)):
        with pytest.raises(ValueError):
            muon_amd.AdamW([p], **bad)
    with pytest.raises(ValueError):
        muon_amd.MuonWithAuxAdam([dict(params=[p], use_muon=False)], adam_state_bits=4)
    with pytest.raises(muon_amd.MuonAmdError):
        muon_amd.AdamW([p]).step()                                # no CPU implementation


def test_tables_are_checked():
    from muon_amd import _lib, plan
    lib = _lib.load()
    d = np.zeros(1, dtype=_lib.ADAMW_DESC)
    d["param"] = d["grad"] = d["exp_avg"] = d["exp_avg_sq"] = 4096
    d["numel"] = 10000
    prefix = plan.adam_block_prefix([10000])
    check = lambda d, prefix, bits: lib.muon_amd_validate_adamw(_lib.host_ptr(d), 1, _lib.host_ptr(prefix), bits)
    assert check(d, prefix, 32) == 0
    assert check(d, prefix, 8) == -1                              # no exponents
    assert check(d, prefix, 16) == -1
    assert check(d, np.array([0, 1], dtype=np.int32), 32) == -1   # blocks that do not cover the tensor
    for name, value in (("param", 0), ("grad", 4098), ("numel", 0), ("dtype", 2)):
        bad = d.copy()
        bad[name] = value
        assert check(bad, prefix, 32) == -1
    assert lib.muon_amd_adamw(None, None, 1, 1, -1, 8, 0.1, 1.0, 0.1, 0.1, 1e-8, 0.5, 0.5, 1, None, None, None) == -1
    assert lib.muon_amd_adamw_values(None, None, 1, 1, None) == -1


@gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_places_beyond_32_bits(bits):
    """A tensor of more than 2^32 elements: the last ones are stepped like those of a small tensor at their place."""
    n, last = 2 ** 32 + 4099, 4096 + 128 * 3
    p = torch.nn.Parameter(torch.zeros(n, dtype=torch.bfloat16, device=DEV))
    p.grad = torch.zeros(n, dtype=torch.bfloat16, device=DEV)
    tail = slice(n - n % SHARED - last, n)
    g = torch.Generator().manual_seed(2)
    p.data[tail] = (torch.randn(p[tail].numel(), generator=g) * 0.05).to(torch.bfloat16).to(DEV)
    p.grad[tail] = (torch.randn(p[tail].numel(), generator=g) * 1e-3).to(torch.bfloat16).to(DEV)
    p.grad[:8] = 1e-3
    small = torch.nn.Parameter(p.detach()[tail].clone())
    small.grad = p.grad[tail].clone()
    opts = [muon_amd.AdamW([q], lr=LR, betas=BETAS, eps=EPS, weight_decay=WD, state_bits=bits) for q in (p, small)]
    for opt in opts:
        opt.step()
    assert torch.equal(p[tail], small)
    if bits == 32:
        assert torch.equal(opts[0].state[p]["exp_avg"][tail], opts[1].state[small]["exp_avg"])
        return
    s = opts[0].state[p]
    gt = small.grad.double().cpu().numpy()
    in32 = lerp32(np.zeros_like(gt), gt, np.float64(np.float32(1 - BETAS[0])))
    E = s["exp_avg_exponent"][tail.start // SHARED:].cpu().numpy()
    np.testing.assert_array_equal(E, shared_exponent(in32, "m"))
    got = np.abs(values(s["exp_avg"][tail].cpu().numpy(), E, "m"))
    lo, hi = (np.abs(rounded(in32, "m", 1, slack, E.astype(np.int64), tail.start)) for slack in (-2.0 ** -16, 2.0 ** -16))
    assert ((got >= lo) & (got <= hi)).all()
    assert (s["exp_avg"][:8] != 0).all() and not s["exp_avg"][8:4096].any()
