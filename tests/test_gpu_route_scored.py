"""Routing by scores with a bias and within groups of experts, against the formulas in 64 bits and against differences (GPU).

The choices have to be those of the definition evaluated in 64 bits, ties at the lowest index.  Bounds of the rest, U = 2^-24: those of
test_gpu_route.py, where a probability is held to 64 U and a weight to 128 U of itself; a sigmoid is nearer (its exponential 4 U, a sum, a reciprocal
and a product 4 U), and the sum of up to 1024 of them adds 32 U.  A gradient adds products of these: 256 U of the sum of the magnitudes of its terms."""
import pytest
import torch

import muon_amd

gpu = pytest.mark.gpu
DEV = "cuda:0"
U = 2.0 ** -24
UNIT = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}
F32, BF16 = torch.float32, torch.bfloat16
INF = float("inf")


def make(shape, k, dtype, seed=0, std=1.5, masked=False, spread=0.1):
    g = torch.Generator().manual_seed(seed)
    logits = (torch.randn(*shape, generator=g) * std).to(dtype)
    mask = torch.rand(*shape[:-1], generator=g) < 0.7 if masked else None
    return logits, mask, torch.randn(*shape[:-1], k, generator=g), torch.randn(shape[-1], generator=g) * spread


def exact(logits, k, scores, bias, groups, kept, mask, normalize, dw, cb, cz):
    x = logits.double().reshape(-1, logits.shape[-1])
    T, E = x.shape
    b = torch.zeros(E, dtype=torch.float64) if bias is None else bias.double()
    can = (x > -INF) & (b > -INF)
    on = torch.ones(T, dtype=torch.bool) if mask is None else mask.reshape(-1)
    on = on & can.any(1)
    n = max(int(on.sum()), 1)
    y = torch.where(on[:, None], x, 0.0)
    p, lse = torch.softmax(y, 1), torch.logsumexp(y, 1)
    s = torch.sigmoid(y) if scores == "sigmoid" else p
    c = torch.where(can, s + b, -INF)
    if kept < groups:
        two = c.view(T, groups, -1).sort(2, descending=True)[0][:, :, :2]
        score = two[:, :, 0] + (torch.where(two[:, :, 1] > -INF, two[:, :, 1], 0.0) if two.shape[2] > 1 else 0.0)
        place = torch.sort(torch.sort(score, dim=1, descending=True, stable=True)[1], dim=1)[1]
        c = torch.where((place < kept).repeat_interleave(E // groups, 1), c, -INF)
    order = torch.sort(c, dim=1, descending=True, stable=True)[1][:, :k]
    there = on[:, None] & (c.gather(1, order) > -INF)
    chosen = torch.where(there, s.gather(1, order), 0.0)
    total = chosen.sum(1, keepdim=True)
    w = chosen / torch.where(total > 0, total, 1.0) if normalize else chosen
    indices = torch.where(there, order, -1)
    counts = torch.bincount(indices[there], minlength=E)
    Z = s.sum(1, keepdim=True)
    Z = torch.where(Z > 0, Z, 1.0)
    share = s / Z * on[:, None]
    balance = E * float((counts.double() / (n * k) * share.sum(0) / n).sum())
    zed = torch.where(on, 2 * cz / n * lse, 0.0)[:, None]
    u = (cb * E * counts.double() / (n * k) / n)[None, :] * on[:, None]
    dw = torch.where(there, dw.double().reshape(T, k), 0.0)
    ds, mag = (u - (share * u).sum(1, keepdim=True)) / Z, (u.abs() + (share * u.abs()).sum(1, keepdim=True)) / Z
    inner, outer = ((dw - (dw * w).sum(1, keepdim=True)), dw.abs() + (dw.abs() * w).sum(1, keepdim=True)) if normalize else (dw, dw.abs())
    per = torch.where(total > 0, 1 / total, 0.0) if normalize else torch.ones_like(total)
    ds = ds.scatter_add(1, order, torch.where(there, inner * per, 0.0))
    mag = mag.scatter_add(1, order, torch.where(there, outer * per, 0.0))
    if scores == "sigmoid":
        dl, mag = s * (1 - s) * ds, s * (1 - s) * mag
    else:
        dl, mag = p * (ds - (p * ds).sum(1, keepdim=True)), p * (mag + (p * mag).sum(1, keepdim=True))
    return dict(weights=w, indices=indices, counts=counts, balance=balance, z=float((torch.where(on, lse, 0.0) ** 2).sum() / n), lse=lse[on],
                grad=torch.where(on[:, None], dl + zed * p, 0.0), mag=mag + (zed * p).abs(), tokens=T)


def check(logits, mask, dw, bias, k, scores="sigmoid", groups=1, kept=None, normalize=True, cb=0.3, cz=0.02, layout=lambda t: t):
    leaf = layout(logits.to(DEV)).detach().requires_grad_()
    m, b = (None if t is None else t.to(DEV) for t in (mask, bias))
    r = muon_amd.route_topk(leaf, k, mask=m, normalize=normalize, scores=scores, bias=b, groups=groups, groups_kept=kept)
    grad, = torch.autograd.grad((r.weights, r.balance_loss, r.z_loss), leaf, (dw.to(DEV), torch.tensor(cb, device=DEV), torch.tensor(cz, device=DEV)))
    want = exact(logits, k, scores, bias, groups, groups if kept is None else kept, mask, normalize, dw, cb, cz)
    T, E = want["tokens"], logits.shape[-1]
    assert r.weights.shape == r.indices.shape == logits.shape[:-1] + (k,) and r.counts.shape == (E,)
    assert r.weights.dtype == F32 and r.indices.dtype == torch.int32 and r.counts.dtype == torch.int32 and grad.dtype == logits.dtype
    assert torch.equal(r.indices.cpu().reshape(T, k).long(), want["indices"])
    assert torch.equal(r.counts.cpu().long(), want["counts"])
    w = r.weights.detach().cpu().double().reshape(T, k)
    assert ((w - want["weights"]).abs() <= 128 * U * want["weights"] + 1e-37).all()
    sums = (T / 64 + 256) * U
    assert abs(float(r.balance_loss.detach()) - want["balance"]) <= sums * want["balance"]
    most = float(want["lse"].abs().max()) if len(want["lse"]) else 0.0
    assert abs(float(r.z_loss.detach()) - want["z"]) <= (sums + 4 * U) * want["z"] + 128 * U * most
    off = (grad.cpu().double().reshape(T, E) - want["grad"]).abs() - 256 * U * want["mag"] - UNIT[logits.dtype] * want["grad"].abs()
    assert off.max() <= 1e-37
    return r, grad


SHAPES = [(1, 1), (2, 1), (4, 2), (6, 3), (8, 4), (8, 8), (12, 4), (16, 4), (24, 2), (32, 8), (33, 3), (48, 16), (60, 5), (64, 8), (64, 64), (72, 8), (128, 8),
          (160, 8), (200, 40), (256, 8), (256, 64), (257, 1), (320, 10), (384, 6), (512, 8), (1000, 20), (1024, 8), (1024, 64)]


@gpu
@pytest.mark.parametrize("scores", ["softmax", "sigmoid"])
@pytest.mark.parametrize("experts,groups", SHAPES)
def test_experts_and_groups(experts, groups, scores):
    each = experts // groups
    for kept in sorted({1, (groups + 1) // 2, groups}):
        for dtype in (F32, BF16):
            k = min(kept * each, 8 if dtype == F32 else 3)
            logits, mask, dw, bias = make((37, experts), k, dtype, seed=experts + kept, masked=dtype == BF16)
            check(logits, mask, dw, bias, k, scores, groups, kept, normalize=kept != 1)
            check(logits, mask, dw, None, k, scores, groups, kept)


@gpu
@pytest.mark.parametrize("experts,k,groups,kept", [(8, 8, 1, 1), (8, 7, 2, 2), (16, 16, 4, 4), (40, 32, 2, 2), (64, 32, 8, 4), (1024, 32, 32, 1), (300, 31, 3, 3)])
@pytest.mark.parametrize("scores", ["softmax", "sigmoid"])
def test_many_choices(experts, k, groups, kept, scores):
    logits, mask, dw, bias = make((50, experts), k, F32, seed=k)
    for b in (bias, None):
        check(logits, mask, dw, b, k, scores, groups, kept)


@gpu
@pytest.mark.parametrize("tokens", [1, 2, 63, 257, 5000, 40001])
@pytest.mark.parametrize("experts,k,groups,kept", [(16, 2, 4, 2), (128, 6, 8, 3)])
def test_tokens(tokens, experts, k, groups, kept):
    for dtype, scores in ((BF16, "sigmoid"), (F32, "softmax")):
        logits, mask, dw, bias = make((tokens, experts), k, dtype, seed=tokens, masked=True)
        check(logits, mask, dw, bias, k, scores, groups, kept)


@gpu
@pytest.mark.parametrize("scores", ["softmax", "sigmoid"])
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("groups,kept", [(1, 1), (6, 2)])
def test_ties(dtype, scores, groups, kept):
    g = torch.Generator().manual_seed(1)
    logits = torch.randint(-2, 3, (200, 48), generator=g).to(dtype)
    logits[torch.rand(200, 48, generator=g) < 0.1] = -0.0
    logits[5] = 1.0
    dw = torch.randn(200, 6, generator=g)
    for bias in (None, torch.zeros(48), torch.randint(-1, 2, (48,), generator=g) * 0.25):
        check(logits, None, dw, bias, 6, scores, groups, kept)


@gpu
@pytest.mark.parametrize("scores", ["softmax", "sigmoid"])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_choices_that_32_bits_cannot_tell(dtype, scores):
    """Biases that lift every expert's score to about the same c: what is left between them is below fp32's step."""
    g = torch.Generator().manual_seed(2)
    row = (torch.randn(64, generator=g) * 1.5).to(dtype)
    s = torch.sigmoid(row.double()) if scores == "sigmoid" else torch.softmax(row.double(), 0)
    bias = (0.75 - s).float()
    logits = row.repeat(100, 1)
    dw = torch.randn(100, 6, generator=g)
    spread = (s + bias.double()).max() - (s + bias.double()).min()
    assert 0 < spread < 2.0 ** -23                               # (the biases are rounded to fp32)
    for groups, kept in ((1, 1), (8, 3), (32, 5)):
        check(logits, None, dw, bias, 6, scores, groups, kept)
    # only some rows, between others that are clear
    logits = torch.where((torch.arange(100) % 7 == 0)[:, None], logits, (torch.randn(100, 64, generator=g) * 1.5).to(dtype))
    for groups, kept in ((1, 1), (8, 3)):
        check(logits, None, dw, bias, 6, scores, groups, kept)


@gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_saturated_scores(dtype):
    """Sigmoids that are 1 or 0 in fp32 and differ in 64 bits, with and without biases."""
    g = torch.Generator().manual_seed(3)
    logits = torch.cat([17 + 4 * torch.rand(60, 32, generator=g), -120 + 10 * torch.rand(60, 32, generator=g), -88 - 30 * torch.rand(60, 32, generator=g)]).to(dtype)
    dw = torch.randn(180, 4, generator=g)
    for bias in (None, torch.zeros(32), torch.randn(32, generator=g)):
        r = muon_amd.route_topk(logits.to(DEV), 4, scores="sigmoid", bias=None if bias is None else bias.to(DEV), groups=4, groups_kept=2)
        want = exact(logits, 4, "sigmoid", bias, 4, 2, None, True, dw, 0.0, 0.0)
        assert torch.equal(r.indices.cpu().long(), want["indices"])
        # (beyond the smallest normal number a score is zero, and a row of nothing else has no weights)
        ok = ((r.weights.cpu().double() - want["weights"]).abs() <= 128 * U * want["weights"] + 1e-37).all(1) | (logits.amax(1) < -80)
        assert ok.all() and torch.isfinite(r.weights).all()


@gpu
@pytest.mark.parametrize("scores", ["softmax", "sigmoid"])
@pytest.mark.parametrize("groups,kept", [(1, 1), (8, 3)])
def test_unavailable_experts(scores, groups, kept):
    g = torch.Generator().manual_seed(4)
    logits, mask, dw, bias = make((200, 48), 6, F32, masked=True)
    logits[torch.rand(200, 48, generator=g) < 0.5] = -INF
    logits[7] = -INF                                             # nothing available
    logits[8] = -INF
    logits[8, 40] = 0.25                                         # one expert for six choices
    logits[9, 6:] = -INF                                         # one group
    bias[[3, 17, 18]] = -INF
    mask[[7, 8, 9]] = True
    r, grad = check(logits, mask, dw, bias, 6, scores, groups, kept)
    assert (r.indices[7] == -1).all() and not grad[7].any() and r.indices[8].tolist() == [40] + [-1] * 5 and r.weights[8, 0] == 1
    assert not torch.isin(r.indices.cpu(), torch.tensor([3, 17, 18])).any()
    bias[:] = -INF                                               # none for anybody
    r, grad = check(logits, mask, dw, bias, 6, scores, groups, kept)
    assert (r.indices == -1).all() and not r.weights.any() and float(r.balance_loss) == 0 and not grad.any()


@gpu
@pytest.mark.parametrize("scores", ["softmax", "sigmoid"])
def test_biases_of_any_size(scores):
    logits, mask, dw, bias = make((100, 64), 6, BF16)
    bias[::5] = torch.finfo(F32).min                             # switched off by the type's lowest number
    bias[1::5] = 1000.0
    bias[2::5] = -1000.0
    for groups, kept in ((1, 1), (8, 4), (32, 16)):
        check(logits, mask, dw, bias, 6, scores, groups, kept)


@gpu
@pytest.mark.parametrize("scores", ["softmax", "sigmoid"])
@pytest.mark.parametrize("groups,kept", [(1, 1), (4, 2)])
def test_masked_rows_and_rows_that_are_no_number(scores, groups, kept):
    logits, mask, dw, bias = make((120, 32), 4, F32, masked=True)
    clean, cg = check(logits, mask, dw, bias, 4, scores, groups, kept)
    dirty = logits.clone()
    dirty[~mask] = float("nan")
    again, dg = check(torch.where(mask[:, None], dirty, 0.0), mask, dw, bias, 4, scores, groups, kept)
    leaf = dirty.to(DEV).requires_grad_()
    r = muon_amd.route_topk(leaf, 4, mask=mask.to(DEV), scores=scores, bias=bias.to(DEV), groups=groups, groups_kept=kept)
    for a, b in zip(clean, r):
        assert torch.equal(a, b)
    g, = torch.autograd.grad((r.weights, r.balance_loss, r.z_loss), leaf, (dw.to(DEV), torch.tensor(0.3, device=DEV), torch.tensor(0.02, device=DEV)))
    assert torch.equal(g, cg)

    logits[11, 5] = float("nan")
    leaf = logits.to(DEV).requires_grad_()
    r = muon_amd.route_topk(leaf, 4, scores=scores, bias=bias.to(DEV), groups=groups, groups_kept=kept)
    rest = torch.arange(120) != 11
    assert torch.isnan(r.weights[11]).any() and torch.isfinite(r.weights[rest]).all() and torch.isnan(r.z_loss)
    assert scores == "softmax" or r.indices[11, 0] == 5
    g, = torch.autograd.grad(r.weights, leaf, dw.to(DEV))
    assert torch.isnan(g[11]).any() and torch.isfinite(g[rest]).all()


@gpu
def test_strides_dimensions_and_addresses():
    for dtype in (F32, BF16):
        l, m, dw, b = make((3, 5, 40), 4, dtype, masked=True)
        check(l, m, dw, b, 4, groups=5, kept=2)
        l, m, dw, b = make((33, 50), 4, dtype, masked=True)
        kw = dict(k=4, groups=5, kept=3)
        check(l, m, dw, b, layout=lambda t: torch.cat([t, t[:, :7]], 1)[:, :50], **kw)
        check(l, m, dw, b, layout=lambda t: t.t().contiguous().t(), **kw)
        check(l, m, dw, torch.stack([b, b], 1)[:, 0], **kw)
        for offset in (1, 3):
            def layout(t):
                buf = torch.zeros(t.numel() + 8, dtype=dtype, device=DEV)
                buf[offset:offset + t.numel()] = t.reshape(-1)
                return buf[offset:offset + t.numel()].view(t.shape)
            check(l, m, dw, b, layout=layout, **kw)


@gpu
def test_the_plain_choice_is_what_it_was():
    for dtype in (F32, BF16):
        l, m, dw, _ = make((500, 64), 6, dtype, masked=True)
        a = muon_amd.route_topk(l.to(DEV), 6, mask=m.to(DEV))
        b = muon_amd.route_topk(l.to(DEV), 6, mask=m.to(DEV), scores="softmax", groups=8, groups_kept=8)
        for x, y in zip(a, b):
            assert torch.equal(x, y)
        c = muon_amd.route_topk(l.to(DEV), 6, mask=m.to(DEV), bias=torch.zeros(64, device=DEV))
        assert torch.equal(a.indices, c.indices) and torch.equal(a.counts, c.counts)
        # a bias of a tenth for all changes nothing but what is compared
        d = muon_amd.route_topk(l.to(DEV), 6, mask=m.to(DEV), scores="sigmoid")
        assert torch.equal(a.indices, d.indices)


@gpu
@pytest.mark.parametrize("scores", ["softmax", "sigmoid"])
@pytest.mark.parametrize("normalize", [True, False])
def test_gradient_against_differences(scores, normalize):
    logits, mask, dw, bias = make((6, 12), 3, F32, masked=True)
    _, grad = check(logits, mask, dw, bias, 3, scores, 4, 2, normalize)
    d = torch.randn(6, 12, generator=torch.Generator().manual_seed(4)).double()
    base = exact(logits, 3, scores, bias, 4, 2, mask, normalize, dw, 0, 0)
    counts, n = base["counts"].double(), max(int(mask.sum()), 1)

    def value(x):                                                # (the choice and the counts are constants of the gradient)
        s = torch.sigmoid(x) if scores == "sigmoid" else torch.softmax(x, 1)
        chosen = s.gather(1, base["indices"].clamp(min=0)) * mask[:, None]
        w = chosen / chosen.sum(1, keepdim=True).clamp(min=1e-30) if normalize else chosen
        share = s / s.sum(1, keepdim=True) * mask[:, None]
        z = ((torch.logsumexp(x, 1) * mask) ** 2).sum() / n
        return float((w * dw).sum() + 0.3 * 12 * (counts / (n * 3) * share.sum(0) / n).sum() + 0.02 * z)

    slope = (value(logits.double() + 1e-4 * d) - value(logits.double() - 1e-4 * d)) / 2e-4
    assert abs(float((grad.cpu().double() * d).sum()) - slope) <= 1e-5


@gpu
def test_repeats_streams_and_graphs():
    logits, mask, dw, bias = make((20000, 160), 5, BF16, masked=True)
    first = check(logits, mask, dw, bias, 5, "sigmoid", 8, 3)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = check(logits, mask, dw, bias, 5, "sigmoid", 8, 3)
    torch.cuda.synchronize()
    for a, b in zip((*first[0], first[1]), (*again[0], again[1])):
        assert torch.equal(a, b)
    leaf, b, up = logits.to(DEV).requires_grad_(), bias.to(DEV), dw.to(DEV)

    def step():
        r = muon_amd.route_topk(leaf, 5, scores="sigmoid", bias=b, groups=8, groups_kept=3)
        return (*(t.detach() for t in r), torch.autograd.grad(r.weights, leaf, up)[0])

    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    for round in range(3):
        with torch.no_grad():
            leaf.copy_(logits.to(DEV).roll(round, 0))
            b.mul_(-1.5)
        graph.replay()
        torch.cuda.synchronize()
        for x, y in zip(captured, step()):
            assert torch.equal(x, y)


@gpu
def test_refusals_on_the_device():
    z = torch.zeros(4, 8, device=DEV)
    b = torch.zeros(8, device=DEV)
    for bad in (dict(scores="tanh"), dict(scores=None), dict(groups=0), dict(groups=3), dict(groups=2.0), dict(groups=16), dict(groups=True), dict(groups=4, groups_kept=0),
                dict(groups=4, groups_kept=5), dict(groups=8, groups_kept=1), dict(groups=4, groups_kept="1"), dict(bias=b[:7]), dict(bias=b[None]),
                dict(bias=b.clone().requires_grad_())):
        with pytest.raises(ValueError):
            muon_amd.route_topk(z, 2, **bad)
    with pytest.raises(TypeError):
        muon_amd.route_topk(z, 2, bias=b.bfloat16())
    with pytest.raises(muon_amd.MuonAmdError):
        muon_amd.route_topk(z, 2, bias=b.cpu())
    with pytest.raises(ValueError):
        muon_amd.route_topk(torch.zeros(2, 256, device=DEV), 2, groups=128)
    with torch.no_grad():                                        # (a parameter may hold it where no gradient is recorded)
        muon_amd.route_topk(z, 2, bias=b.clone().requires_grad_())


def test_refusals():
    import ctypes

    from muon_amd import _lib
    with pytest.raises(muon_amd.MuonAmdError):
        muon_amd.route_topk(torch.zeros(4, 8), 2, scores="sigmoid")
    lib = _lib.load()
    good = dict(logits=4096, weights=4096, indices=4096, counts=4096, balance=4096, z=4096, part=4096, lse=4096, lse_rest=4096, partials=4096, dlogits=4096,
                tokens=1, ld_logits=8, experts=8, k=2)
    args = ctypes.byref(_lib.RouteArgs(**good))
    for scores, groups, kept in ((2, 1, 1), (-1, 1, 1), (0, 0, 1), (0, 3, 1), (0, 2, 0), (0, 2, 3), (0, 8, 1), (1, 65, 65)):
        assert lib.muon_amd_route_scored(args, scores, None, groups, kept, None) == -1
    assert lib.muon_amd_route_scored_backward(args, 2, None) == -1
    for bad in (dict(tokens=0), dict(experts=2000), dict(k=9), dict(logits=None), dict(partials=None)):
        assert lib.muon_amd_route_scored(ctypes.byref(_lib.RouteArgs(**{**good, **bad})), 1, None, 1, 1, None) == -1
    assert lib.muon_amd_route_scored_backward(ctypes.byref(_lib.RouteArgs(**{**good, "dlogits": None})), 1, None) == -1
    assert lib.muon_amd_route_scored(None, 1, None, 1, 1, None) == -1 and lib.muon_amd_route_scored_backward(None, 1, None) == -1
    assert lib.muon_amd_route_max_groups() == 64


@gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("scores,values", [("sigmoid", (18.0, 18.25, 19.0, 20.0)), ("softmax", (0.0, -2.0 ** -28, -2.0 ** -27, -2.0 ** -26))])
@pytest.mark.parametrize("experts", [8, 16, 40, 64, 100, 256, 320, 1000])
def test_equal_logits_beside_near_ones(experts, scores, values, dtype):
    """Scores that are one number in 32 bits, of logits of which several are equal and others are not: the equal ones are no reason to stop looking."""
    g = torch.Generator().manual_seed(experts)
    for k in sorted({1, 2, min(8, experts // 2), min(32, experts)}):
        logits, mask, dw, bias = make((41, experts), k, dtype, seed=k)
        near = torch.rand(41, experts, generator=g) < (torch.arange(41)[:, None] + 1) / 41            # from a few of them to all
        pick = torch.tensor(values)[torch.randint(len(values), (41, experts), generator=g)]
        logits = torch.where(near, pick, logits.float() - 12).to(dtype)
        check(logits, mask, dw, None, k, scores)
        # (groups by softmax: 1 + e^-2a is larger than 2 e^-a by a^2, at a = 2^-28 half of 2^-56 of the sum, which 64 bits do not hold)
        if scores == "sigmoid" and experts % 8 == 0 and k <= experts // 8 * 3:
            check(logits, mask, dw, None, k, scores, groups=8, kept=3)
    row = torch.full((1, experts), -30.0)
    row[0, :3] = torch.tensor([values[1], values[1], values[0] if scores == "softmax" else values[2]])
    r, _ = check(row.to(dtype), None, torch.ones(1, 1), None, 1, scores)
    assert r.indices.item() == 2


@gpu
@pytest.mark.parametrize("scores", ["softmax", "sigmoid"])
@pytest.mark.parametrize("experts,k,groups,kept", [(8, 2, 1, 1), (8, 4, 2, 1), (8, 8, 1, 1), (60, 6, 5, 2), (160, 6, 8, 3), (256, 8, 8, 4), (256, 32, 8, 4), (1024, 32, 16, 2)])
def test_rows_of_equal_logits(experts, k, groups, kept, scores):
    for dtype in (F32, BF16):
        logits, mask, dw, bias = make((37, experts), k, dtype, seed=k, masked=True)
        logits[:20] = 0.0
        logits[20:30] = logits[20:30, :1]
        logits[3, ::3] = -INF
        logits[4, 1:] = -INF
        logits[5, 1:experts // groups] = -INF
        logits[25, -1] += 0.5
        logits[26, experts // 2:] -= 0.5
        for b in (None, torch.zeros(experts), torch.full((experts,), 0.25), bias, torch.where(bias > 0.1, -INF, 0.0)):
            check(logits, mask, dw, b, k, scores, groups, kept)


@gpu
@pytest.mark.parametrize("scores", ["softmax", "sigmoid"])
def test_offsets_beyond_32_bits(scores):
    tokens, experts = 2 ** 31 // 256 + 5, 256
    logits = torch.zeros(tokens, experts, dtype=BF16, device=DEV)
    tail, _, dw, bias = make((999, experts), 8, BF16, seed=1)
    logits[-999:] = tail.to(DEV)
    leaf, alone = logits.requires_grad_(), tail.to(DEV).requires_grad_()
    r, s = (muon_amd.route_topk(t, 8, scores=scores, bias=bias.to(DEV), groups=8, groups_kept=4) for t in (leaf, alone))
    assert torch.equal(r.indices[-999:], s.indices) and torch.equal(r.weights[-999:], s.weights)
    assert int(r.counts.sum()) == 8 * tokens
    give = torch.zeros(tokens, 8, device=DEV)
    give[-999:] = dw.to(DEV)
    got, = torch.autograd.grad(r.weights, leaf, give)
    want, = torch.autograd.grad(s.weights, alone, dw.to(DEV))
    assert torch.equal(got[-999:], want) and not got[:-999].any()
