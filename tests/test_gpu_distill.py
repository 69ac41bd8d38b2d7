"""Distillation from top logits, its loss and gradient, against the formulas in 64 bits and against differences (GPU).

Bounds.  U = 2^-24, u the output type's unit roundoff.  With y = (x - max) / T in units of ln 2, the kernels' exponent is off by
2 U |y| (the factor log2(e) / T) and U |y| (its rounding), the power by 2 U: (3 |y| + 4) U relative to itself, with |y| <= Y
over what the test holds.  The sum of V of them adds a rounding for every 256th, one for every pack of four, and 64 for the joins:
E = (3 Y + 4 + V / 128 + 64) U bounds log p absolutely and p relative to itself, and log q, q likewise with the list in
the place of V.  A term q (log q - log p) is off by q (2 E + E |log q - log p| + 4 U (|log q| + |log p|)), and a sum of K terms by 64 U and 2 U K of its
magnitudes.  A gradient T g (p - q) is off by |T g| (p + q) (E + 4 U), and by u of itself."""
import math

import pytest
import torch

import muon_amd

gpu = pytest.mark.gpu
DEV = "cuda:0"
U = 2.0 ** -24
UNIT = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}
F32, BF16 = torch.float32, torch.bfloat16
INF = float("inf")


def make(shape, vocab, k, dtype, seed=0, std=2.0, masked=False, index=torch.int64, teacher=None):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(*shape, vocab, generator=g) * std).to(dtype)
    v = (torch.randn(*shape, k, generator=g) * std + 3).to(teacher or dtype)
    i = torch.argsort(torch.rand(*shape, vocab, generator=g), -1)[..., :k] if vocab >= k else torch.randint(vocab, (*shape, k), generator=g)
    mask = torch.rand(*shape, generator=g) < 0.7 if masked else None
    return x, v, i.to(index), mask


def exact(x, v, i, mask, T, up):
    """losses, gradient for upstream `up` of each token (or a number for the mean), and the bounds of both."""
    V, K = x.shape[-1], v.shape[-1]
    x, v, i = x.double().reshape(-1, V), v.double().reshape(-1, K), i.long().reshape(-1, K)
    there = (i >= 0) & (i < V) & (v > -INF)
    on = there.any(1) if mask is None else there.any(1) & mask.reshape(-1)
    n = max(int(on.sum()), 1)
    x = torch.where(on[:, None], x, 0.0)
    at = i.clamp(0, V - 1)
    t = torch.where(there, v / T, -INF)
    t = torch.where(there.any(1, keepdim=True), t, 0.0)
    logq, logp = torch.log_softmax(t, 1), torch.log_softmax(x / T, 1)
    q = torch.where(there & on[:, None], logq.exp(), 0.0)
    lp = logp.gather(1, at)
    diff = torch.where(q > 0, logq - lp, 0.0)
    losses = T * T * (q * diff).sum(1)
    Y = max(float((y.amax(1, keepdim=True) - y)[y > -INF].max()) for y in (x / T, t)) / math.log(2)
    E = (3 * Y + 4 + max(V, K) / 128 + 64) * U
    mags = torch.where(q > 0, q * (2 * E + E * diff.abs() + 4 * U * (logq.abs() + lp.abs())), 0.0).sum(1)
    loss_off = T * T * (mags + (64 + 2 * K) * U * (q * diff.abs()).sum(1))
    g = (torch.full((len(x),), up / n) if isinstance(up, float) else up.double().reshape(-1)) * T
    g = torch.where(on, g.double(), 0.0)[:, None]
    p = logp.exp() * on[:, None]
    spread = torch.zeros_like(p).scatter_add_(1, at, q)
    grad = g * (p - spread)
    return dict(on=on, n=n, losses=losses, loss_off=loss_off, grad=grad, grad_off=g.abs() * (p + spread) * (E + 4 * U))


def check(x, v, i, mask=None, T=1.0, layout=lambda t: t, reduction="mean", up=0.7):
    leaf = layout(x.to(DEV)).detach().requires_grad_()
    m = None if mask is None else mask.to(DEV)
    give = torch.randn(x.shape[:-1], generator=torch.Generator().manual_seed(9)) if reduction == "none" else torch.tensor(up)
    loss = muon_amd.distill_topk(leaf, v.to(DEV), i.to(DEV), temperature=T, mask=m, reduction=reduction)
    grad, = torch.autograd.grad(loss, leaf, give.to(DEV))
    want = exact(x, v, i, mask, T, give if reduction == "none" else (up if reduction == "mean" else torch.full(x.shape[:-1], up)))
    assert loss.dtype == F32 and grad.dtype == x.dtype and grad.shape == x.shape
    got = loss.detach().cpu().double()
    if reduction == "none":
        assert got.shape == x.shape[:-1]
        assert ((got.reshape(-1) - want["losses"]).abs() <= want["loss_off"] + U * want["losses"].abs()).all()
    else:
        n = want["n"] if reduction == "mean" else 1
        tokens = len(want["losses"])
        bound = (want["loss_off"].sum() + (tokens / 256 + 32) * U * want["losses"].abs().sum()) / n
        assert got.dim() == 0 and abs(float(got) - float(want["losses"].sum() / n)) <= float(bound)
    off = (grad.cpu().double().reshape(want["grad"].shape) - want["grad"]).abs() - want["grad_off"] - UNIT[x.dtype] * want["grad"].abs()
    assert off.max() <= 1e-37
    return loss.detach(), grad


@gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("vocab", [1, 2, 7, 8, 9, 63, 1000, 4096, 4097, 8191, 16384, 32768, 32771, 50257])
def test_vocabularies(vocab, dtype):
    for k in sorted({1, min(5, vocab), min(64, vocab)}):
        check(*make((3,), vocab, k, dtype, seed=vocab + k))


@gpu
@pytest.mark.parametrize("tokens", [1, 2, 5, 257, 1025])
def test_tokens(tokens):
    check(*make((tokens,), 5003, 8, BF16, seed=tokens, masked=True, index=torch.int32))


@gpu
@pytest.mark.parametrize("k", [1, 2, 63, 64, 65, 200, 1024])
def test_lists(k):
    check(*make((4,), 3000, k, F32, seed=k))
    check(*make((4,), 17, k, F32, seed=k))                       # most indices several times


@gpu
@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
@pytest.mark.parametrize("T", [0.5, 1, 3.0, 20.0])
def test_temperatures_and_reductions(T, reduction):
    check(*make((2, 9), 1234, 6, BF16, masked=True), T=T, reduction=reduction)
    check(*make((2, 9), 1234, 6, F32, teacher=BF16), T=T, reduction=reduction)
    check(*make((18,), 1234, 6, BF16, teacher=F32), T=T, reduction=reduction)


@gpu
def test_entries_that_are_not_there():
    x, v, i, _ = make((40,), 700, 6, F32)
    g = torch.Generator().manual_seed(3)
    i[torch.rand(40, 6, generator=g) < 0.3] = -1
    i[4], i[5] = -1, 700                                         # (beyond the vocabulary: not there either)
    i[6] = torch.tensor([1 << 40, -5, 699, 0, -1, 700])
    v[torch.rand(40, 6, generator=g) < 0.2] = -INF
    v[7] = -INF
    loss, grad = check(x, v, i, reduction="none")
    assert loss[4] == 0 and loss[5] == 0 and loss[7] == 0 and not grad[[4, 5, 7]].any()
    check(x, v, i)
    check(x, v, i, T=2.0, reduction="sum")
    x[4], x[5] = float("nan"), INF                               # logits of tokens that take no part are not read
    loss, grad = muon_amd.distill_topk(x.to(DEV), v.to(DEV), i.to(DEV)), None
    assert torch.isfinite(loss)
    check(x, v, i)


@gpu
def test_nothing_takes_part():
    x, v, i, _ = make((5,), 100, 3, BF16)
    for mask, index in ((torch.zeros(5, dtype=torch.bool), i), (None, torch.full_like(i, -1))):
        loss, grad = check(x, v, index, mask)
        assert loss == 0 and not grad.any()
    for reduction, shape in (("mean", ()), ("none", (0,))):
        empty = torch.zeros(0, 100, device=DEV, requires_grad=True)
        loss = muon_amd.distill_topk(empty, torch.zeros(0, 3, device=DEV), torch.zeros(0, 3, dtype=torch.int32, device=DEV), reduction=reduction)
        assert loss.shape == shape and not loss.detach().any()
        loss.sum().backward()
        assert empty.grad.shape == (0, 100)


@gpu
def test_masked_rows_may_hold_anything():
    x, v, i, mask = make((50,), 900, 4, F32, masked=True)
    clean = check(x, v, i, mask)
    x[~mask], v[~mask], i[~mask] = float("nan"), float("nan"), 1 << 33
    dirty = check(x, v, i, mask)
    assert torch.equal(clean[0], dirty[0]) and torch.equal(clean[1], dirty[1])


@gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_logits_that_are_infinite_or_no_number(dtype):
    x, v, i, _ = make((20,), 300, 4, dtype)
    ban = torch.rand(20, 300, generator=torch.Generator().manual_seed(2)) < 0.5
    ban.scatter_(1, i, False)
    x[ban] = -INF                                                # a vocabulary with words masked out
    _, grad = check(x, v, i)
    assert not grad[ban].any()
    x[3, i[3, 0]] = -INF                                         # the student cannot say what the teacher does
    x[5, 7] = float("nan")
    x[6, 7] = INF
    x[7] = -INF
    v[8, 1] = float("nan")
    leaf = x.to(DEV).requires_grad_()
    loss = muon_amd.distill_topk(leaf, v.to(DEV), i.to(DEV), reduction="none")
    grad, = torch.autograd.grad(loss.sum(), leaf)
    bad = torch.tensor([3, 5, 6, 7, 8])
    rest = torch.tensor([r for r in range(20) if r not in bad])
    assert loss[3] == INF and torch.isnan(loss[[5, 6, 7, 8]]).all() and torch.isfinite(loss[rest]).all()
    assert torch.isfinite(grad[3]).all() and all(torch.isnan(grad[r]).any() for r in (5, 6, 7, 8)) and torch.isfinite(grad[rest]).all()


@gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("at", [-1e30, -65280.0, 1e4, 1e30])
def test_logits_far_from_zero(at, dtype):
    """All of a row's logits at one value: every probability is 1 / V, however coarse the type is there."""
    V, K = 1000, 4
    x = torch.full((3, V), at, dtype=dtype)
    v = torch.full((3, K), at, dtype=dtype)
    i = torch.arange(K).repeat(3, 1)
    leaf = x.to(DEV).requires_grad_()
    loss = muon_amd.distill_topk(leaf, v.to(DEV), i.to(DEV), reduction="sum")
    grad, = torch.autograd.grad(loss, leaf)
    assert abs(float(loss) - 3 * math.log(V / K)) <= 3 * 200 * U * math.log(V)
    want = torch.full((3, V), 1 / V, dtype=torch.float64)
    want[:, :K] -= 1 / K
    assert ((grad.cpu().double() - want).abs() <= (UNIT[dtype] + 200 * U) * want.abs() + 200 * U / V).all()


@gpu
def test_strides_dimensions_and_addresses():
    for dtype in (F32, BF16):
        x, v, i, mask = make((3, 5), 203, 4, dtype, masked=True)
        check(x, v, i, mask)
        check(x, v, i, mask, reduction="none")
        x, v, i, mask = make((15,), 203, 4, dtype, masked=True)
        check(x, v, i, mask, layout=lambda t: torch.cat([t, t[:, :9]], 1)[:, :203])
        check(x, v, i, mask, layout=lambda t: t.t().contiguous().t())
        for offset in (1, 3):
            def layout(t):
                buf = torch.zeros(t.numel() + 8, dtype=dtype, device=DEV)
                buf[offset:offset + t.numel()] = t.reshape(-1)
                return buf[offset:offset + t.numel()].view(t.shape)
            check(x, v, i, mask, layout=layout)
        wide = torch.randn(15, 12).to(dtype)
        check(x, wide[:, ::3], torch.arange(12).repeat(15, 1)[:, ::3])
        one = torch.randn(203).to(dtype)
        check(one, v[0], i[0], reduction="none")                 # a token by itself


@gpu
def test_rows_next_to_the_outputs_stay():
    """The gradient of a leaf that is part of a larger buffer is written within its own rows."""
    x, v, i, _ = make((7,), 1001, 5, BF16)
    _, a = check(x, v, i)
    _, b = check(x, v, i, layout=lambda t: torch.cat([t, t], 1)[:, :1001])
    assert torch.equal(a, b)


@gpu
@pytest.mark.parametrize("T", [1.0, 2.5])
def test_gradient_against_differences(T):
    x, v, i, mask = make((5,), 40, 3, F32, masked=True)
    _, grad = check(x, v, i, mask, T=T, up=1.0)
    d = torch.randn(5, 40, generator=torch.Generator().manual_seed(4)).double()

    def value(y):
        r = exact(y, v, i, mask, T, 1.0)
        return float(r["losses"].sum() / r["n"])

    slope = (value(x.double() + 1e-4 * d) - value(x.double() - 1e-4 * d)) / 2e-4
    assert abs(float((grad.cpu().double() * d).sum()) - slope) <= 1e-5


@gpu
def test_a_student_that_equals_its_teacher():
    """Over the whole vocabulary as its list, the loss is zero and so is the gradient, to rounding."""
    x = torch.randn(6, 500, generator=torch.Generator().manual_seed(1))
    loss, grad = check(x, x, torch.arange(500).repeat(6, 1), T=1.5)
    assert abs(float(loss)) <= 1e-5


@gpu
def test_repeats_streams_and_graphs():
    x, v, i, mask = make((300,), 20011, 9, BF16, masked=True)
    first = check(x, v, i, mask)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = check(x, v, i, mask)
    torch.cuda.synchronize()
    assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])

    leaf = x.to(DEV).requires_grad_()
    args = v.to(DEV), i.to(DEV)
    m = mask.to(DEV)

    def step():
        return torch.autograd.grad(muon_amd.distill_topk(leaf, *args, mask=m), leaf, torch.tensor(0.7, device=DEV) if not torch.cuda.is_current_stream_capturing() else up)[0]

    up = torch.tensor(0.7, device=DEV)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for scale in (1.0, 0.5, 2.0):
        with torch.no_grad():
            leaf.copy_((x * scale).to(DEV))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, step())


@gpu
def test_offsets_beyond_32_bits():
    tokens, vocab = 2 ** 31 // 40000 + 7, 40000
    x = torch.zeros(tokens, vocab, dtype=BF16, device=DEV)
    small, v, i, _ = make((9,), vocab, 5, BF16)
    x[-9:] = small.to(DEV)
    index = torch.full((tokens, 5), -1, dtype=torch.int32, device=DEV)
    values = torch.zeros(tokens, 5, dtype=BF16, device=DEV)
    index[-9:], values[-9:] = i.to(DEV).int(), v.to(DEV)
    want, wgrad = check(small, v, i, up=1.0)
    leaf = x.requires_grad_()
    loss = muon_amd.distill_topk(leaf, values, index, reduction="none")
    assert not loss[:-9].any()
    grad, = torch.autograd.grad(loss[-9:].mean(), leaf)
    assert abs(float(loss.sum() / 9) - float(want)) <= 64 * U * float(want)
    assert (grad[-9:].float() - wgrad.float()).abs().max() <= 2.0 ** -7 * wgrad.float().abs().max()
    assert not grad[-10].any() and not grad[0].any()


@gpu
def test_gradients_stop_where_they_should():
    x, v, i, _ = (t if t is None else t.to(DEV) for t in make((4,), 50, 3, F32))
    assert not muon_amd.distill_topk(x, v, i).requires_grad
    with torch.no_grad():
        assert not muon_amd.distill_topk(x.requires_grad_(), v, i).requires_grad
    loss = muon_amd.distill_topk(x, v, i)
    g, = torch.autograd.grad(loss, x, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(g.sum(), x)
    with pytest.raises(ValueError):
        muon_amd.distill_topk(x, v.requires_grad_(), i)


@gpu
def test_refusals_on_the_device():
    x, v, i, _ = (t if t is None else t.to(DEV) for t in make((4,), 50, 3, F32))
    for bad in (dict(temperature=0.0), dict(temperature=-1.0), dict(temperature=INF), dict(temperature=float("nan")), dict(temperature="1"),
                dict(reduction="max"), dict(reduction=None), dict(mask=torch.ones(4, device=DEV)), dict(mask=torch.ones(3, dtype=torch.bool, device=DEV))):
        with pytest.raises(ValueError):
            muon_amd.distill_topk(x, v, i, **bad)
    for args in ((x, v[:3], i[:3]), (x, v, i[:, :2]), (x, v[:, :0], i[:, :0]), (x, v[0], i[0]),
                 (x, torch.zeros(4, 1025, device=DEV), torch.zeros(4, 1025, dtype=torch.int32, device=DEV)), (x[:, :0], v, i)):
        with pytest.raises(ValueError):
            muon_amd.distill_topk(*args)
    for args in ((x.half(), v, i), (x, v.half(), i), (x, v, i.float()), (x, v, i.short())):
        with pytest.raises(TypeError):
            muon_amd.distill_topk(*args)
    for args in ((x, v.cpu(), i), (x, v, i.cpu())):
        with pytest.raises(muon_amd.MuonAmdError):
            muon_amd.distill_topk(*args)


def test_refusals():
    import ctypes

    from muon_amd import _lib
    with pytest.raises(muon_amd.MuonAmdError):
        muon_amd.distill_topk(torch.zeros(4, 8), torch.zeros(4, 2), torch.zeros(4, 2, dtype=torch.int32))     # no CPU implementation
    lib = _lib.load()
    pointers = ("logits", "teacher", "indices", "losses", "part", "stats", "partials", "counter", "dloss", "dlogits")
    good = dict({p: 4096 for p in pointers}, tokens=1, ld_logits=8, ld_teacher=2, ld_indices=2, vocab=8, top=2, index_bits=32, temperature=1.0)
    for bad in (dict(tokens=0), dict(tokens=1 << 25), dict(vocab=0), dict(vocab=(1 << 30) + 1), dict(top=0), dict(top=1025), dict(dtype=5), dict(teacher_dtype=2), dict(index_bits=16),
                dict(reduction=3), dict(temperature=0.0), dict(temperature=INF), dict(logits=None), dict(teacher=None), dict(indices=None), dict(stats=None)):
        for call in (lib.muon_amd_distill, lib.muon_amd_distill_backward):
            assert call(ctypes.byref(_lib.DistillArgs(**{**good, **bad})), None) == -1
    for name in ("losses", "partials", "counter"):
        assert lib.muon_amd_distill(ctypes.byref(_lib.DistillArgs(**{**good, name: None})), None) == -1
    for name in ("dloss", "dlogits"):
        assert lib.muon_amd_distill_backward(ctypes.byref(_lib.DistillArgs(**{**good, name: None})), None) == -1
    assert lib.muon_amd_distill_backward(ctypes.byref(_lib.DistillArgs(**{**good, "tokens": 1 << 24, "vocab": 1 << 30})), None) == -1
    assert lib.muon_amd_distill(None, None) == -1 and lib.muon_amd_distill_backward(None, None) == -1
    assert lib.muon_amd_distill_partials(0, 8, 0) == 0 and lib.muon_amd_distill_partials(100, 8, 0) > 0


@gpu
def test_the_largest_temperature():
    check(*make((5,), 1234, 6, F32), T=1e15)
    check(*make((5,), 1234, 6, F32), T=1e15, reduction="none")


@gpu
def test_the_smallest_temperature():
    # p and q have one entry each: a loss is T (max - x at the teacher's best), of a difference's rounding and those of 1 / T, log2(e), T ^ 2, ln 2
    # and four products, twelve in all; the gradient is T g at the one and - T g at the other.
    T = 1e-15
    x, v, i, _ = make((5,), 1234, 6, F32)
    leaf = x.to(DEV).requires_grad_()
    losses = muon_amd.distill_topk(leaf, v.to(DEV), i.to(DEV), temperature=T, reduction="none")
    grad, = torch.autograd.grad(losses.sum(), leaf)
    at, top = i.gather(1, v.argmax(1, keepdim=True)), x.argmax(1, keepdim=True)
    want = T * (x.double().gather(1, top) - x.double().gather(1, at))[:, 0]
    assert ((losses.cpu().double() - want).abs() <= 12 * U * want).all()
    one = torch.zeros(5, 1234, dtype=torch.float64)
    expected = one.scatter(1, top, T) - one.scatter(1, at, T)
    assert ((grad.cpu().double() - expected).abs() <= 12 * U * T).all()


@gpu
def test_refusals_of_temperatures():
    x, v, i, _ = (t if t is None else t.to(DEV) for t in make((4,), 50, 3, F32))
    for T in (1e-16, 1e16, 10 ** 20):
        with pytest.raises(ValueError):
            muon_amd.distill_topk(x, v, i, temperature=T)


def test_refusals_beyond_a_launch():
    import ctypes

    from muon_amd import _lib
    lib = _lib.load()
    pointers = ("logits", "teacher", "indices", "losses", "part", "stats", "partials", "counter", "dloss", "dlogits")
    good = dict({p: 4096 for p in pointers}, tokens=1 << 24, ld_logits=8, ld_teacher=2, ld_indices=2, vocab=8, top=2, index_bits=32, temperature=1.0)
    for bad in ({}, dict(vocab=1 << 30), dict(tokens=1, temperature=1e-16), dict(tokens=1, temperature=1e16)):      # 2^24 workgroups of 256: 2^32 threads
        for call in (lib.muon_amd_distill, lib.muon_amd_distill_backward):
            assert call(ctypes.byref(_lib.DistillArgs(**{**good, **bad})), None) == -1
