"""Cross entropy of a linear head, its logsumexps and gradients, against the formulas in 64 bits and against differences (GPU).

Bounds.  U = 2^-24, u = 2^-8 (bf16).  Most inputs here are whole multiples of a power of two, so small that every logit is exact
in fp32 whatever the order of its sum (test_random_values has the others: D U sum |h w| more for each logit).  With y = x - max in
units of ln 2, the exponent is off by 2 U |y|, the power by 2 U, and a sum of V powers in the kernels' order by (V / 256 + 128) U: E = (3 Y + V / 256 + 136) U
bounds lse absolutely beside U |lse| and p relative to itself.  loss adds U (|lse| + |x|).  The logits' gradient e = (g + z) p - g [target] is off by
(E + 4 U) (|g + z| p) + 4 U |g| [target], and by u of itself when it is rounded; dh = e W and dW = e^T h by the product of that with |W|, |h|, by
(V + 64) U and (N + 64) U of the product of the magnitudes (sums in any order), and by u of themselves.  Those are worst cases of
sums whose terms are rounded independently, so the norms of the errors are held too: sqrt(2) u of ||e|| ... is what one rounding of each term and one of
the result leave, relative to the norm of the result, if they are all of half a step; 2 u is allowed."""
import math

import pytest
import torch

import muon_amd

gpu = pytest.mark.gpu
DEV = "cuda:0"
U, u = 2.0 ** -24, 2.0 ** -8
BF16 = torch.bfloat16
IGNORE = -100


def make(n, v, d, seed=0, ignored=0.0, index=torch.int64):
    """Hidden states and a matrix whose products are whole multiples of a power of two, with logits of a spread of about 2."""
    g = torch.Generator().manual_seed(seed)
    h = torch.randint(-3, 4, (n, d), generator=g).to(BF16)
    scale = 2.0 ** -round(math.log2(4.6 * 2.0 * d ** 0.5 / 2))
    w = (torch.randint(-8, 9, (v, d), generator=g) * scale).to(BF16)
    t = torch.randint(v, (n,), generator=g)
    t[torch.rand(n, generator=g) < ignored] = IGNORE
    return h, w, t.to(index)


def exact(h, w, t, gl, gz, ignore=IGNORE, inexact=False):
    """losses, lse, gradients (on the GPU, in 64 bits) with the bounds of each; gl, gz: gradients of each token's loss and lse."""
    h, w, t = h.to(DEV).double(), w.to(DEV).double(), t.to(DEV).long()
    n, v, d = len(h), len(w), h.shape[1]
    on = t != ignore
    h = torch.where(on[:, None], h, 0.0)
    at = torch.where(on, t, 0)[:, None]
    x = h @ w.t()
    dx = d * U * (h.abs() @ w.abs().t()) if inexact else torch.zeros(1, 1, dtype=torch.float64, device=DEV)
    lse = torch.logsumexp(x, 1)
    Y = float((x.amax(1, keepdim=True) - x).max()) / math.log(2)
    E = (3 * Y + v / 256 + 136) * U + 2 * dx.amax(1)
    loss = torch.where(on, lse - x.gather(1, at)[:, 0], 0.0)
    loss_off = torch.where(on, E + dx.amax(1) + 2 * U * (lse.abs() + x.gather(1, at)[:, 0].abs()), 0.0)
    gl, gz = torch.where(on, gl.to(DEV).double(), 0.0)[:, None], torch.where(on, gz.to(DEV).double(), 0.0)[:, None]
    p = (x - lse[:, None]).exp()
    hit = torch.zeros_like(p).scatter_(1, at, 1.0)
    e = (gl + gz) * p - gl * hit
    off = (E[:, None] + 4 * U) * (gl + gz).abs() * p + 4 * U * gl.abs() * hit + u * e.abs()
    out = dict(on=on, loss=loss, loss_off=loss_off, lse=torch.where(on, lse, 0.0), lse_off=torch.where(on, E + 2 * U * lse.abs(), 0.0))
    out["dh"], out["dw"] = e @ w, e.t() @ h
    out["dh_off"] = off @ w.abs() + (v + 64) * U * (e.abs() @ w.abs()) + u * out["dh"].abs()
    out["dw_off"] = off.t() @ h.abs() + (n + 64) * U * (e.abs().t() @ h.abs()) + u * out["dw"].abs()
    # per row of the products: what roundings of half a step leave in the norms
    out["dh_norm"] = u * ((e ** 2) @ (w ** 2)).sum().sqrt() + u * out["dh"].norm()
    out["dw_norm"] = u * ((e ** 2).t() @ (h ** 2)).sum().sqrt() + u * out["dw"].norm()
    return out


def check(h, w, t, reduction="mean", lay_h=lambda a: a, lay_w=lambda a: a, z=True, ignore=IGNORE, inexact=False, shape=None):
    hd, wd = lay_h(h.to(DEV)).detach().requires_grad_(), lay_w(w.to(DEV)).detach().requires_grad_()
    td = t.to(DEV)
    n = len(t)
    g = torch.Generator().manual_seed(7)
    gz = torch.randn(n, generator=g) / n if z else torch.zeros(n)
    up = torch.randn(n, generator=g) if reduction == "none" else torch.tensor(0.75)
    taking = max(int((t != ignore).sum()), 1)
    gl = up if reduction == "none" else torch.full((n,), 0.75 / (taking if reduction == "mean" else 1), dtype=torch.float64)
    if shape:
        hd, td = hd.view(*shape, -1), td.view(shape)
        out = muon_amd.linear_cross_entropy(hd, wd, td, reduction=reduction, ignore_index=ignore)
        assert out.lse.shape == shape and out.loss.shape == (shape if reduction == "none" else ())
    else:
        out = muon_amd.linear_cross_entropy(hd, wd, td, reduction=reduction, ignore_index=ignore)
    assert out.loss.dtype == out.lse.dtype == torch.float32
    outs, ups = [out.loss], [up.to(DEV).view(out.loss.shape)]
    if z:
        outs, ups = outs + [out.lse], ups + [gz.to(DEV).view(out.lse.shape)]
    dh, dw = torch.autograd.grad(outs, (hd, wd), ups)
    want = exact(h, w, t, gl, gz, ignore, inexact)
    loss, lse = out.loss.detach().double().reshape(-1), out.lse.detach().double().reshape(-1)
    assert ((lse - want["lse"]).abs() <= want["lse_off"]).all()
    if reduction == "none":
        assert ((loss - want["loss"]).abs() <= want["loss_off"]).all()
    else:
        per = taking if reduction == "mean" else 1
        bound = (want["loss_off"].sum() + (n / 1024 + 64) * U * want["loss"].abs().sum()) / per
        assert abs(float(loss - want["loss"].sum() / per)) <= float(bound)
    for name, got in (("dh", dh), ("dw", dw)):
        assert got.dtype == BF16
        got = got.double().reshape(want[name].shape)
        assert ((got - want[name]).abs() <= want[name + "_off"] + 1e-37).all(), name
        assert (got - want[name]).norm() <= 2 * want[name + "_norm"] + 1e-37, name
    return out.loss.detach(), out.lse.detach(), dh, dw


@gpu
@pytest.mark.parametrize("tokens", [1, 2, 15, 16, 17, 32, 33, 63, 64])
@pytest.mark.parametrize("width", [64, 200])
def test_few_tokens(tokens, width):
    check(*make(tokens, 1000, width, seed=tokens))


@gpu
@pytest.mark.parametrize("tokens", [31, 32, 33, 64])
def test_few_tokens_of_a_large_matrix(tokens):
    check(*make(tokens, 33000, 512, seed=tokens, ignored=0.2))   # (between the two ways that few tokens go)
    check(*make(tokens, 33000, 520, seed=tokens, ignored=0.2), reduction="none")


@gpu
@pytest.mark.parametrize("tokens", [65, 127, 128, 129, 255, 256, 257, 511, 700])
def test_tokens(tokens):
    check(*make(tokens, 1111, 128, seed=tokens, ignored=0.2))


@gpu
@pytest.mark.parametrize("vocab", [1, 2, 3, 63, 64, 65, 127, 128, 129, 255, 256, 257, 300, 1000, 5003])
@pytest.mark.parametrize("tokens", [5, 150])
def test_vocabularies(vocab, tokens):
    check(*make(tokens, vocab, 64, seed=vocab, index=torch.int32))


@gpu
@pytest.mark.parametrize("width", [1, 2, 7, 8, 9, 31, 32, 56, 63, 64, 65, 100, 127, 128, 192, 256, 320, 500, 1024, 1600])
@pytest.mark.parametrize("tokens", [3, 130])
def test_widths(width, tokens):
    check(*make(tokens, 700, width, seed=width))


@gpu
def test_large_tiles():
    check(*make(2100, 16700, 128, ignored=0.1))
    check(*make(1500, 22000, 72))


@gpu
def test_pieces_of_the_vocabulary():
    check(*make(8200, 65600, 64, ignored=0.3))
    check(*make(300, 65600, 64))


@gpu
@pytest.mark.parametrize("tokens", [40, 300])
@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
def test_reductions_and_shapes(reduction, tokens):
    for z in (False, True):
        check(*make(tokens, 900, 64, ignored=0.3), reduction=reduction, z=z)
    check(*make(tokens, 900, 64, ignored=0.3), reduction=reduction, shape=(tokens // 10, 10))
    check(*make(1, 900, 64), reduction=reduction, shape=())


@gpu
@pytest.mark.parametrize("tokens", [50, 500])
def test_ignored_tokens_may_hold_anything(tokens):
    h, w, t = make(tokens, 800, 128, ignored=0.5)
    clean = check(h, w, t)
    h[t == IGNORE] = float("nan")
    h[t.argmin()] = float("inf")
    dirty = check(h, w, t)
    for a, b in zip(clean, dirty):
        assert torch.equal(a, b)
    assert not dirty[2][(t == IGNORE).to(DEV)].any()
    t7 = torch.where(t == IGNORE, 7, torch.where(t == 7, 8, t))
    other = check(h, w, t7, ignore=7)
    assert not other[2][(t7 == 7).to(DEV)].any()


@gpu
@pytest.mark.parametrize("tokens", [1, 50, 500])
def test_nothing_takes_part(tokens):
    h, w, t = make(tokens, 300, 64)
    t[:] = IGNORE
    loss, lse, dh, dw = check(h, w, t)
    assert loss == 0 and not lse.any() and not dh.any() and not dw.any()


@gpu
def test_no_tokens():
    w = torch.zeros(10, 8, dtype=BF16, device=DEV, requires_grad=True)
    h = torch.zeros(0, 8, dtype=BF16, device=DEV, requires_grad=True)
    for reduction in ("mean", "none"):
        out = muon_amd.linear_cross_entropy(h, w, torch.zeros(0, dtype=torch.int64, device=DEV), reduction=reduction)
        assert out.lse.shape == (0,) and not out.loss.detach().any()
        dh, dw = torch.autograd.grad(out.loss.sum(), (h, w))
        assert dh.shape == (0, 8) and not dw.any()


@gpu
@pytest.mark.parametrize("tokens", [20, 200])
@pytest.mark.parametrize("bad", [-1, 400, 1 << 40, -(1 << 33)])
def test_targets_outside_of_the_vocabulary(bad, tokens):
    h, w, t = make(tokens, 400, 64)
    t[3] = bad
    hd, wd = h.to(DEV).requires_grad_(), w.to(DEV).requires_grad_()
    out = muon_amd.linear_cross_entropy(hd, wd, t.to(DEV), reduction="none")
    rest = torch.arange(tokens) != 3
    assert torch.isnan(out.loss[3]) and torch.isfinite(out.loss[rest]).all() and torch.isfinite(out.lse).all()
    dh, dw = torch.autograd.grad(out.loss.sum(), (hd, wd))
    assert torch.isnan(dh[3]).all() and torch.isfinite(dh[rest]).all() and torch.isnan(dw).any()


@gpu
@pytest.mark.parametrize("tokens", [20, 200])
def test_numbers_that_are_none(tokens):
    h, w, t = make(tokens, 400, 64)
    h[5, 3] = float("nan")
    h[6, 3] = float("inf")
    hd = h.to(DEV).requires_grad_()
    out = muon_amd.linear_cross_entropy(hd, w.to(DEV), t.to(DEV), reduction="none")
    rest = torch.tensor([i for i in range(tokens) if i not in (5, 6)])
    assert torch.isnan(out.loss[[5, 6]]).all() and torch.isfinite(out.loss[rest]).all()
    dh, = torch.autograd.grad(out.loss.sum(), hd)
    assert torch.isnan(dh[[5, 6]]).any(1).all() and torch.isfinite(dh[rest]).all()


@gpu
@pytest.mark.parametrize("tokens", [10, 140])
@pytest.mark.parametrize("at", [1e4, -1e4, 3e7])
def test_logits_far_from_zero(at, tokens):
    """All logits of a token at one value far from zero: every probability is 1 / V."""
    v, d = 1000, 64
    h = torch.zeros(tokens, d, dtype=BF16)
    w = torch.zeros(v, d, dtype=BF16)
    h[:, 0], w[:, 0] = at, 1.0
    t = torch.arange(tokens)
    hd, wd = h.to(DEV).requires_grad_(), w.to(DEV).requires_grad_()
    out = muon_amd.linear_cross_entropy(hd, wd, t.to(DEV), reduction="sum")
    dh, dw = torch.autograd.grad(out.loss, (hd, wd))
    # (the loss is the logarithm of V beside the difference of two equal numbers)
    value = abs(float(hd[0, 0].detach()))
    assert abs(float(out.loss.detach()) - tokens * math.log(v)) <= tokens * (200 * U * math.log(v) + U * math.log(v) + 2 * U * value * (math.log(v) / value < 1))
    hits = torch.bincount(t, minlength=v).double()
    want = (tokens / v - hits) * float(hd[0, 0].detach())
    assert ((dw[:, 0].double().cpu() - want).abs() <= 3 * u * ((tokens / v + hits) * value)).all()


@gpu
@pytest.mark.parametrize("tokens", [30, 300])
def test_strides_and_addresses(tokens):
    h, w, t = make(tokens, 333, 64, ignored=0.2)

    def offset(by):
        def lay(a):
            buf = torch.zeros(a.numel() + 16, dtype=BF16, device=DEV)
            buf[by:by + a.numel()] = a.reshape(-1)
            return buf[by:by + a.numel()].view(a.shape)
        return lay

    def wide(by):
        return lambda a: torch.cat([a, torch.full_like(a[:, :by], float("nan"))], 1)[:, :a.shape[1]]

    plain = check(h, w, t)
    for lay in (offset(1), offset(8), wide(3), wide(8), wide(64), lambda a: a.t().contiguous().t()):
        for kw in (dict(lay_h=lay), dict(lay_w=lay)):
            other = check(h, w, t, **kw)
            for a, b in zip(plain, other):
                assert torch.equal(a, b)
    one = torch.randint(-3, 4, (1, 64), generator=torch.Generator().manual_seed(1)).to(BF16)
    check(one.expand(tokens, 64), w, t, lay_h=lambda a: one.to(DEV).expand(tokens, 64))         # one hidden state for all


@gpu
@pytest.mark.parametrize("tokens,vocab,width", [(1, 5000, 2048), (64, 3000, 777), (300, 4000, 512), (1111, 3003, 1600)])
def test_random_values(tokens, vocab, width):
    g = torch.Generator().manual_seed(5)
    h = torch.randn(tokens, width, generator=g).to(BF16)
    w = (torch.randn(vocab, width, generator=g) * 2 / width ** 0.5).to(BF16)
    check(h, w, torch.randint(vocab, (tokens,), generator=g), inexact=True)


@gpu
def test_gradients_against_differences():
    h, w, t = make(30, 50, 16, ignored=0.2)
    _, _, dh, dw = check(h, w, t, z=False)
    g = torch.Generator().manual_seed(4)
    a, b = torch.randn(h.shape, generator=g).double(), torch.randn(w.shape, generator=g).double()

    def value(s):
        x = (h.double() + s * a) @ (w.double() + s * b).t()
        return float(0.75 * torch.nn.functional.cross_entropy(x, t))

    slope = (value(1e-5) - value(-1e-5)) / 2e-5
    got = float((dh.double().cpu() * a).sum() + (dw.double().cpu() * b).sum())
    # (two roundings of each term of the two sums)
    assert abs(got - slope) <= 3 * u * float((dh.double().cpu() * a).abs().sum() + (dw.double().cpu() * b).abs().sum())


@gpu
def test_one_gradient_alone():
    for tokens in (40, 300):
        h, w, t = make(tokens, 600, 128, ignored=0.1)
        _, _, dh, dw = check(h, w, t, z=False)
        for i in range(2):
            hd, wd = h.to(DEV).requires_grad_(i == 0), w.to(DEV).requires_grad_(i == 1)
            out = muon_amd.linear_cross_entropy(hd, wd, t.to(DEV))
            got, = torch.autograd.grad(out.loss, (hd, wd)[i], torch.tensor(0.75, device=DEV))
            assert torch.equal(got, (dh, dw)[i])
        hd = h.to(DEV).requires_grad_()
        out = muon_amd.linear_cross_entropy(hd, w.to(DEV), t.to(DEV))
        z, = torch.autograd.grad(out.lse.sum(), hd)              # through the logsumexps alone
        p = torch.softmax(h.to(DEV).double() @ w.to(DEV).double().t(), 1) * (t != IGNORE).to(DEV)[:, None]
        assert ((z.double() - p @ w.to(DEV).double()).abs() <= 3 * u * (p @ w.to(DEV).double().abs())).all()


@gpu
def test_single_tokens_and_batches_agree():
    """What a token gets does not go by how many others there are, beyond the rounding of its sums."""
    h, w, t = make(300, 2000, 256)
    args = w.to(DEV)
    all_ = muon_amd.linear_cross_entropy(h.to(DEV), args, t.to(DEV), reduction="none")
    for i in (0, 150, 299):
        one = muon_amd.linear_cross_entropy(h[i].to(DEV), args, t[i].to(DEV), reduction="none")
        assert abs(float(one.loss - all_.loss[i])) <= 300 * U * (1 + float(one.lse))


@gpu
def test_repeats_streams_and_graphs():
    for tokens in (20, 700):
        h, w, t = make(tokens, 3000, 192, ignored=0.2)
        first = check(h, w, t)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            again = check(h, w, t)
        torch.cuda.synchronize()
        for a, b in zip(first, again):
            assert torch.equal(a, b)

        hd, wd, td = h.to(DEV).requires_grad_(), w.to(DEV).requires_grad_(), t.to(DEV)
        one = torch.ones((), device=DEV)

        def step():
            out = muon_amd.linear_cross_entropy(hd, wd, td)
            return (out.loss.detach(), *torch.autograd.grad(out.loss, (hd, wd), one))

        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step()
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            captured = step()
        for round in range(3):                                   # other values and another number of tokens in each
            with torch.no_grad():
                hd.copy_((h * (1 + round)).to(DEV))
                td.copy_(t.to(DEV).roll(round))
                td[:5 * round] = IGNORE
            graph.replay()
            torch.cuda.synchronize()
            for a, b in zip(captured, step()):
                assert torch.equal(a, b)


@gpu
def test_offsets_beyond_32_bits():
    """A matrix of more than 2^32 bytes and 2^31 elements."""
    v, d, n = 2 ** 31 // 4096 + 300, 4096, 70
    w = torch.zeros(v, d, dtype=BF16, device=DEV)
    g = torch.Generator().manual_seed(3)
    w[-200:] = (torch.randint(-8, 9, (200, d), generator=g) / 256).to(BF16).to(DEV)
    h = torch.randint(-3, 4, (n, d), generator=g).to(BF16).to(DEV)
    t = torch.randint(v - 200, v, (n,), generator=g).to(DEV)
    x = h.double() @ w[-200:].double().t()
    lse = torch.logaddexp(torch.logsumexp(x, 1), torch.full((n,), math.log(v - 200), dtype=torch.float64, device=DEV))
    loss = lse - x.gather(1, (t - (v - 200))[:, None])[:, 0]
    off = (3 * 60 + v / 256 + 200) * U * (1 + lse.abs())
    wd = w.requires_grad_()
    for rows in (n, 8):
        out = muon_amd.linear_cross_entropy(h[:rows], wd, t[:rows], reduction="none")
        assert ((out.loss.detach() - loss[:rows]).abs() <= off[:rows]).all()
    dw, = torch.autograd.grad(out.loss.sum(), wd)
    p = (x[:8] - lse[:8, None]).exp()
    hit = torch.zeros_like(p).scatter_(1, (t[:8] - (v - 200))[:, None], 1.0)
    want = (p - hit).t() @ h[:8].double()
    assert ((dw[-200:].double() - want).abs() <= 3 * u * ((p + hit).t() @ h[:8].double().abs())).all()
    low = (-lse[:8]).exp() @ h[:8].double()
    assert ((dw[:1000].double() - low).abs() <= 3 * u * ((-lse[:8]).exp() @ h[:8].double().abs())).all()


@gpu
def test_gradients_stop_where_they_should():
    h, w, t = (a.to(DEV) for a in make(70, 100, 64))
    assert not muon_amd.linear_cross_entropy(h, w, t).loss.requires_grad
    out = muon_amd.linear_cross_entropy(h.requires_grad_(), w, t)
    assert out.loss.requires_grad and out.lse.requires_grad
    g, = torch.autograd.grad(out.loss, h, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(g.float().sum(), h)


@gpu
def test_refusals_on_the_device():
    h, w, t = (a.to(DEV) for a in make(4, 10, 8))
    for args in ((h, w[:, :4], t), (h, w[0], t), (h, w, t[:3]), (h[:, :0], w[:, :0], t), (h, w[:0], t), (h, w, t[:, None])):
        with pytest.raises(ValueError):
            muon_amd.linear_cross_entropy(*args)
    for kw in (dict(reduction="max"), dict(reduction=1), dict(ignore_index=1.5), dict(ignore_index=1 << 70), dict(ignore_index=True)):
        with pytest.raises(ValueError):
            muon_amd.linear_cross_entropy(h, w, t, **kw)
    for args in ((h.float(), w, t), (h, w.float(), t), (h, w, t.float()), (h.half(), w, t)):
        with pytest.raises(TypeError):
            muon_amd.linear_cross_entropy(*args)
    for args in ((h, w.cpu(), t), (h, w, t.cpu()), (h.cpu(), w, t)):
        with pytest.raises(muon_amd.MuonAmdError):
            muon_amd.linear_cross_entropy(*args)


def test_refusals():
    import ctypes

    from muon_amd import _lib
    with pytest.raises(muon_amd.MuonAmdError):
        muon_amd.linear_cross_entropy(torch.zeros(4, 8, dtype=BF16), torch.zeros(5, 8, dtype=BF16), torch.zeros(4, dtype=torch.int64))
    lib = _lib.load()
    pointers = ("hidden", "weight", "targets", "losses", "lse", "part", "order", "rows", "stats", "counter", "workspace", "dhidden", "dweight")
    good = dict({p: 4096 for p in pointers}, tokens=100, ld_hidden=8, ld_weight=8, width=8, vocab=10, target_bits=32, workspace_bytes=1 << 40)
    calls = lib.muon_amd_head_loss, lib.muon_amd_head_loss_backward
    for bad in (dict(tokens=0), dict(tokens=(1 << 24) + 1), dict(width=0), dict(width=(1 << 16) + 1), dict(vocab=0), dict(vocab=(1 << 24) + 1), dict(target_bits=8), dict(reduction=5),
                dict(workspace=4100), dict(ld_weight=1 << 30), dict(ld_weight=-1), dict(workspace_bytes=100), dict(hidden=None), dict(weight=None), dict(targets=None),
                dict(order=None), dict(rows=None), dict(stats=None), dict(part=None), dict(workspace=None)):
        for call in calls:
            assert call(ctypes.byref(_lib.HeadLossArgs(**{**good, **bad})), None) == -1, bad
    for name in ("losses", "lse", "counter"):
        assert lib.muon_amd_head_loss(ctypes.byref(_lib.HeadLossArgs(**{**good, name: None})), None) == -1
    assert lib.muon_amd_head_loss_backward(ctypes.byref(_lib.HeadLossArgs(**{**good, "dhidden": None, "dweight": None})), None) == -1
    for call in calls:
        assert call(None, None) == -1
    for backward in (0, 1):
        assert lib.muon_amd_head_loss_workspace(ctypes.byref(_lib.HeadLossArgs(**good)), backward) > 0
        assert lib.muon_amd_head_loss_workspace(None, backward) == 0


@gpu
@pytest.mark.parametrize("tokens", [1020, 1023, 1024, 1025])
def test_around_a_thousand_tokens(tokens):
    check(*make(tokens, 500, 72, seed=tokens, ignored=0.4))      # (between the two ways that tokens are numbered)
    check(*make(tokens, 500, 64, seed=tokens), z=False)


@gpu
@pytest.mark.parametrize("tokens", [1, 16, 17, 32, 33, 48, 64])
@pytest.mark.parametrize("vocab,width", [(1, 64), (65, 1216), (200, 1990), (640, 4160), (7, 130)])
def test_streamed_matrices(tokens, vocab, width):
    check(*make(tokens, vocab, width, seed=tokens + vocab, ignored=0.3))         # (blocks of 64 channels: one, numbers that are no multiple of the waves', part of one)


@gpu
def test_few_tokens_and_large_tiles_of_the_matrix():
    check(*make(70, 66000, 2050, seed=1, ignored=0.2))           # (the matrix's gradient in tiles that are many for a k-block or two)
