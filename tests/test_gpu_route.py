"""Routing of tokens to experts with its losses and gradients against the formulas in 64 bits and against differences (GPU).

Bounds.  U = 2^-24, u the output type's unit roundoff.  Logits differ by less than 24 from their row's largest here: the
difference takes one rounding (24 U in the exponential's argument), the exponential 4 U, a sum of positive terms over at
most 16 in sequence and 6 joins 22 U: 64 U bounds a probability, and twice that a weight, relative to itself.  lse takes 64 U
and its own rounding.  Sums over T tokens add a rounding for each row that a lane adds and for each partial sum: (T / 64 +
256) U of a sum of positive terms.  A gradient adds products of these: 256 U of the sum of the magnitudes of its terms."""
import pytest
import torch

import muon_amd

gpu = pytest.mark.gpu
DEV = "cuda:0"
U = 2.0 ** -24
UNIT = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}
F32, BF16 = torch.float32, torch.bfloat16


def make(shape, k, dtype, seed=0, std=1.5, masked=False):
    g = torch.Generator().manual_seed(seed)
    logits = (torch.randn(*shape, generator=g) * std).to(dtype)
    mask = torch.rand(*shape[:-1], generator=g) < 0.7 if masked else None
    dw = torch.randn(*shape[:-1], k, generator=g)
    return logits, mask, dw


def exact(logits, k, mask, normalize, dw, cb, cz):
    x = logits.double().reshape(-1, logits.shape[-1])
    T, E = x.shape
    on = torch.ones(T, dtype=torch.bool) if mask is None else mask.reshape(-1)
    on = on & (x > -torch.inf).any(1)
    n = max(int(on.sum()), 1)
    p = torch.where(on[:, None], torch.softmax(torch.where(on[:, None], x, 0.0), -1), 0.0)
    lse = torch.where(on, torch.logsumexp(torch.where(on[:, None], x, 0.0), -1), 0.0)
    order = torch.sort(x, dim=-1, descending=True, stable=True)[1][:, :k]
    there = on[:, None] & (x.gather(1, order) > -torch.inf)
    indices = torch.where(there, order, -1)
    chosen = torch.where(there, p.gather(1, order), 0.0)
    total = chosen.sum(1, keepdim=True)
    w = chosen / torch.where(total > 0, total, 1.0) if normalize else chosen
    counts = torch.bincount(indices[there], minlength=E)
    balance = E * float((counts.double() / (n * k) * p.sum(0) / n).sum())
    z = float((lse ** 2).sum() / n)
    g = (cb * E * counts.double() / (n * k) / n).expand(T, E)
    dw = torch.where(there, dw.double().reshape(T, k), 0.0)
    add = torch.zeros(T, E, dtype=torch.float64)
    mag = torch.zeros(T, E, dtype=torch.float64)
    if normalize:
        part, pm = w * (dw - (w * dw).sum(1, keepdim=True)), w * (dw.abs() + (w * dw.abs()).sum(1, keepdim=True))
        add.scatter_add_(1, order, torch.where(there, part, 0.0))
        mag.scatter_add_(1, order, torch.where(there, pm, 0.0))
    else:
        g = g.scatter_add(1, order, dw)
    zed = 2 * cz / n * lse[:, None]
    dl = p * (g - (p * g).sum(1, keepdim=True)) + zed * p + add
    mag = mag + p * (g.abs() + (p * g.abs()).sum(1, keepdim=True)) + (zed * p).abs()
    return dict(weights=w, indices=indices, counts=counts, balance=balance, z=z, lse=lse, grad=dl, mag=mag, tokens=T)


def check(logits, k, mask, dw, normalize=True, cb=0.3, cz=0.02, layout=lambda t: t):
    leaf = layout(logits.to(DEV)).detach().requires_grad_()
    m = None if mask is None else mask.to(DEV)
    r = muon_amd.route_topk(leaf, k, mask=m, normalize=normalize)
    grad, = torch.autograd.grad((r.weights, r.balance_loss, r.z_loss), leaf,
                                (dw.to(DEV), torch.tensor(cb, device=DEV), torch.tensor(cz, device=DEV)))
    want = exact(logits, k, mask, normalize, dw, cb, cz)
    assert r.weights.shape == r.indices.shape == logits.shape[:-1] + (k,) and r.counts.shape == logits.shape[-1:]
    assert r.weights.dtype == F32 and r.indices.dtype == torch.int32 and r.counts.dtype == torch.int32
    T, E = want["tokens"], logits.shape[-1]
    assert torch.equal(r.indices.cpu().reshape(T, k).long(), want["indices"])
    assert torch.equal(r.counts.cpu().long(), want["counts"])
    w = r.weights.detach().cpu().double().reshape(T, k)
    assert ((w - want["weights"]).abs() <= 128 * U * want["weights"] + 1e-37).all()
    sums = (T / 64 + 256) * U
    assert abs(float(r.balance_loss.detach()) - want["balance"]) <= sums * want["balance"]
    assert abs(float(r.z_loss.detach()) - want["z"]) <= (sums + 4 * U) * want["z"] + 128 * U * float(want["lse"].abs().max())
    off = (grad.cpu().double().reshape(T, E) - want["grad"]).abs() - 256 * U * want["mag"] - UNIT[logits.dtype] * want["grad"].abs()
    assert grad.dtype == logits.dtype and off.max() <= 1e-37
    return r, grad


@gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("experts", [1, 2, 3, 7, 8, 9, 16, 17, 32, 33, 60, 64, 65, 128, 160, 256, 257, 512, 1000, 1024])
def test_experts(experts, dtype):
    for k in sorted({1, min(2, experts), min(8, experts), min(32, experts)}):
        check(*(lambda l, m, dw: (l, k, m, dw))(*make((37, experts), k, dtype, seed=experts, masked=k == 2)), normalize=k != 8)


@gpu
@pytest.mark.parametrize("tokens", [1, 2, 63, 257, 5000, 40001])
@pytest.mark.parametrize("experts,k", [(8, 2), (24, 4), (128, 6)])
def test_tokens(tokens, experts, k):
    logits, mask, dw = make((tokens, experts), k, BF16, seed=tokens, masked=True)
    check(logits, k, mask, dw)


@gpu
@pytest.mark.parametrize("normalize", [True, False])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_ties_zeros_and_unavailable_experts(dtype, normalize):
    g = torch.Generator().manual_seed(1)
    # few values, so that most choices are ties; both zeros; whole rows of one value; the lowest finite value
    logits = torch.randint(-2, 3, (200, 48), generator=g).to(dtype)
    logits[torch.rand(200, 48, generator=g) < 0.1] = -0.0
    logits[5] = 1.0
    dw = torch.randn(200, 6, generator=g)
    check(logits, 6, None, dw, normalize)
    gone = torch.rand(200, 48, generator=g) < 0.5
    logits = logits.masked_fill(gone, -float("inf"))
    logits[7] = -float("inf")                                    # nothing available
    logits[8] = -float("inf")
    logits[8, 40] = 0.25                                         # one expert for six choices
    logits[9, 3:] = -float("inf")
    r, grad = check(logits, 6, None, dw, normalize)
    assert (r.indices[7] == -1).all() and (r.weights[7] == 0).all() and not grad[7].any()
    assert r.indices[8].tolist() == [40] + [-1] * 5 and r.weights[8, 1:].tolist() == [0.0] * 5
    lowest = torch.full((4, 48), torch.finfo(dtype).min, dtype=dtype)
    lowest[1, 5] = 0.0
    r = muon_amd.route_topk(lowest.to(DEV), 6, normalize=normalize)
    assert r.indices[0].tolist() == [0, 1, 2, 3, 4, 5] and r.indices[1].tolist() == [5, 0, 1, 2, 3, 4]
    assert torch.isfinite(r.weights).all()


@gpu
def test_nothing_takes_part():
    logits, _, dw = make((50, 16), 2, F32)
    for mask in (torch.zeros(50, dtype=torch.bool), None):
        l = logits if mask is not None else torch.full_like(logits, -float("inf"))
        r, grad = check(l, 2, mask, dw)
        assert float(r.balance_loss) == 0 and float(r.z_loss) == 0 and not r.counts.any() and not grad.any()
    r = muon_amd.route_topk(torch.zeros(0, 16, device=DEV, requires_grad=True), 2)
    assert r.weights.shape == (0, 2) and not r.counts.any() and float(r.balance_loss) == 0


@gpu
def test_masked_rows_may_hold_anything():
    logits, mask, dw = make((300, 32), 4, F32, masked=True)
    clean, cg = check(logits, 4, mask, dw)
    dirty = logits.clone()
    dirty[~mask] = float("nan")
    r = muon_amd.route_topk(dirty.to(DEV).requires_grad_(), 4, mask=mask.to(DEV))
    for a, b in zip(clean, r):
        assert torch.equal(a, b)
    leaf = dirty.to(DEV).requires_grad_()
    r = muon_amd.route_topk(leaf, 4, mask=mask.to(DEV))
    g, = torch.autograd.grad(r.balance_loss + r.z_loss, leaf)
    assert torch.isfinite(g).all()


@gpu
def test_nan_shows_and_stays_in_its_row():
    logits, _, dw = make((40, 16), 3, F32)
    logits[11, 5] = float("nan")
    leaf = logits.to(DEV).requires_grad_()
    r = muon_amd.route_topk(leaf, 3)
    assert r.indices[11, 0] == 5 and torch.isnan(r.weights[11]).any() and torch.isnan(r.z_loss)
    assert torch.isfinite(r.weights[torch.arange(40) != 11]).all()
    g, = torch.autograd.grad(r.weights.sum(), leaf)
    assert torch.isnan(g[11]).any() and torch.isfinite(g[torch.arange(40) != 11]).all()


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("normalize", [True, False])
@pytest.mark.parametrize("bad", [float("inf"), float("nan")], ids=["inf", "nan"])
@pytest.mark.parametrize("experts", [8, 48, 200, 300])
def test_rows_whose_softmax_is_not_a_number(experts, bad, normalize, dtype):
    logits = torch.randn(40, experts, generator=torch.Generator().manual_seed(5)).to(dtype)
    clean = logits.clone()
    logits[11, 5] = bad
    x, c = (t.to(DEV).requires_grad_() for t in (logits, clean))
    r, q = (muon_amd.route_topk(t, 3, normalize=normalize) for t in (x, c))
    rest = torch.arange(40) != 11
    assert r.indices[11, 0] == 5 and torch.isnan(r.weights[11]).all() and torch.isnan(r.balance_loss) and not torch.isfinite(r.z_loss)
    assert torch.equal(r.weights[rest], q.weights[rest]) and torch.equal(r.indices[rest], q.indices[rest])
    up = torch.ones_like(r.weights)
    up[:, 0] = 2.0
    g, h = (torch.autograd.grad(t.weights, u, up)[0] for t, u in ((r, x), (q, c)))
    assert torch.isnan(g[11]).all() and torch.equal(g[rest], h[rest])


@gpu
def test_strides_dimensions_and_addresses():
    for dtype in (F32, BF16):
        l, m, dw = make((3, 5, 40), 4, dtype, masked=True)
        check(l, 4, m, dw)
        l, m, dw = make((33, 50), 4, dtype, masked=True)
        check(l, 4, m, dw, layout=lambda t: torch.cat([t, t[:, :7]], 1)[:, :50])
        check(l, 4, m, dw, layout=lambda t: t.t().contiguous().t())
        check(l, 4, m, dw.expand(33, 4))
        for offset in (1, 3):
            def layout(t):
                buf = torch.zeros(t.numel() + 8, dtype=dtype, device=DEV)
                buf[offset:offset + t.numel()] = t.reshape(-1)
                return buf[offset:offset + t.numel()].view(t.shape)
            check(l, 4, m, dw, layout=layout)


@gpu
def test_parts_of_the_gradient():
    logits, mask, dw = make((100, 24), 3, F32, masked=True)
    for names in (["weights"], ["balance_loss"], ["z_loss"]):
        leaf = logits.to(DEV).requires_grad_()
        r = muon_amd.route_topk(leaf, 3, mask=mask.to(DEV))
        give = {"weights": dw.to(DEV), "balance_loss": torch.tensor(0.3, device=DEV), "z_loss": torch.tensor(0.02, device=DEV)}
        got, = torch.autograd.grad([getattr(r, n) for n in names], leaf, [give[n] for n in names])
        want = exact(logits, 3, mask, True, dw if "weights" in names else 0 * dw, 0.3 if "balance_loss" in names else 0.0,
                     0.02 if "z_loss" in names else 0.0)
        assert ((got.cpu().double() - want["grad"]).abs() <= 256 * U * want["mag"] + U * want["grad"].abs() + 1e-37).all()


@gpu
@pytest.mark.parametrize("normalize", [True, False])
def test_gradient_against_differences(normalize):
    logits, mask, dw = make((6, 12), 3, F32, masked=True)
    _, grad = check(logits, 3, mask, dw, normalize)
    d = torch.randn(6, 12, generator=torch.Generator().manual_seed(4)).double()
    counts = exact(logits, 3, mask, normalize, dw, 0, 0)["counts"].double()

    def value(x):                                                # (counts are constants of the gradient)
        r = exact(x, 3, mask, normalize, dw, 0, 0)
        n = max(int(mask.sum()), 1)
        p = torch.softmax(x, -1) * mask[:, None]
        return float((r["weights"] * dw * mask[:, None]).sum() + 0.3 * 12 * (counts / (n * 3) * p.sum(0) / n).sum() + 0.02 * r["z"])

    slope = (value(logits.double() + 1e-4 * d) - value(logits.double() - 1e-4 * d)) / 2e-4
    assert abs(float((grad.cpu().double() * d).sum()) - slope) <= 1e-5


@gpu
def test_repeats_and_streams():
    logits, mask, dw = make((20000, 100), 5, BF16, masked=True)
    first = check(logits, 5, mask, dw)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = check(logits, 5, mask, dw)
    torch.cuda.synchronize()
    for a, b in zip((*first[0], first[1]), (*again[0], again[1])):
        assert torch.equal(a, b)


@gpu
def test_refusals_on_the_device():
    z = torch.zeros(4, 8, device=DEV)
    for bad in (dict(k=0), dict(k=9), dict(k=2.5), dict(k=2, mask=torch.ones(4, device=DEV)), dict(k=2, mask=torch.ones(3, dtype=torch.bool, device=DEV))):
        with pytest.raises(ValueError):
            muon_amd.route_topk(z, **bad)
    with pytest.raises(ValueError):
        muon_amd.route_topk(torch.zeros(2, 1025, device=DEV), 2)
    with pytest.raises(ValueError):
        muon_amd.route_topk(torch.zeros(2, 64, device=DEV), 33)
    with pytest.raises(TypeError):
        muon_amd.route_topk(z.half(), 2)
    with pytest.raises(muon_amd.MuonAmdError):
        muon_amd.route_topk(z, 2, mask=torch.ones(4, dtype=torch.bool))


def test_refusals():
    import ctypes

    from muon_amd import _lib
    with pytest.raises(muon_amd.MuonAmdError):
        muon_amd.route_topk(torch.zeros(4, 8), 2)                # no CPU implementation
    lib = _lib.load()
    good = dict(logits=4096, weights=4096, indices=4096, counts=4096, balance=4096, z=4096, part=4096, lse=4096, partials=4096, dlogits=4096,
                tokens=1, ld_logits=8, experts=8, k=2)
    for bad in (dict(tokens=0), dict(experts=0), dict(experts=2000), dict(k=0), dict(k=9), dict(logits=None), dict(lse=None), dict(dtype=5)):
        for call in (lib.muon_amd_route, lib.muon_amd_route_backward):
            assert call(ctypes.byref(_lib.RouteArgs(**{**good, **bad})), None) == -1
    assert lib.muon_amd_route(ctypes.byref(_lib.RouteArgs(**{**good, "partials": None})), None) == -1
    assert lib.muon_amd_route_backward(ctypes.byref(_lib.RouteArgs(**{**good, "dlogits": None})), None) == -1
    assert lib.muon_amd_route(None, None) == -1 and lib.muon_amd_route_backward(None, None) == -1
    assert lib.muon_amd_route_partials(0, 8) == 0 and lib.muon_amd_route_partials(100, 8) > 0


@gpu
def test_no_second_derivatives():
    leaf = torch.randn(4, 8, device=DEV, requires_grad=True)
    g, = torch.autograd.grad(muon_amd.route_topk(leaf, 2).balance_loss, leaf, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(g.sum(), leaf)


@gpu
def test_offsets_beyond_32_bits():
    """More than 2^31 logits in rows that pass 2^32 elements over the tensor: the last tokens are chosen for as in a small
    call, and the counts are whole."""
    tokens, experts, k = 2 ** 31 // 512 + 5, 512, 2
    wide = torch.zeros(tokens, 2 * experts, dtype=BF16, device=DEV)
    logits = wide[:, :experts]
    small, _, dw = make((40, experts), k, BF16)
    logits[-40:] = small.to(DEV)
    leaf = logits.requires_grad_()
    r = muon_amd.route_topk(leaf, k)
    few = small.to(DEV).requires_grad_()
    want = muon_amd.route_topk(few, k)
    assert torch.equal(r.indices[-40:], want.indices) and torch.equal(r.weights[-40:], want.weights)
    assert (r.indices[:-40] == torch.tensor([0, 1], dtype=torch.int32, device=DEV)).all()
    counts = want.counts.clone()
    counts[:2] += tokens - 40
    assert torch.equal(r.counts, counts)
    grads = torch.zeros(tokens, k, device=DEV)
    grads[-40:] = dw.to(DEV)
    a, = torch.autograd.grad(r.weights, leaf, grads)
    b, = torch.autograd.grad(want.weights, few, dw.to(DEV))
    assert torch.equal(a[-40:], b) and not a[:-40].any()
