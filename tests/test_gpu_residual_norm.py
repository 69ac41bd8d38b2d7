"""The residual step between two blocks and its gradients against the formulas in 64 bits, and against differences (GPU).

Bounds.  With u the unit roundoff of the output's type (2^-24, 2^-8) and U = 2^-24: a row's mean of squares is off by at most
(D / 8 + 10) U of itself if its sums were in sequence, in the worst case; its threads add at most 32 terms each and join
in a tree, so 48 U covers it, and half of that goes into the norm's factor.  h takes it on the part that is added, y on
itself; the sigmoid is off by 8 U.  With m the sum of the magnitudes of the terms of an output, 96 U m + u |output| bounds
each; the gradients go by two reductions (c1, c2) and take twice that, with the means' terms in magnitude in m.  A sum over T
rows adds a rounding for each row that a thread adds (rows of one workgroup in sequence): (T / 64 + 96) U of the sum of magnitudes."""
import pytest
import torch

import muon_amd

gpu = pytest.mark.gpu
DEV = "cuda:0"
U = 2.0 ** -24
UNIT = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}
EPS = 1e-6
F32, BF16 = torch.float32, torch.bfloat16


def make(shape, stream=BF16, block=BF16, weights=BF16, gate="channel", scale="channel", seed=0, xstd=2.0):
    g = torch.Generator().manual_seed(seed)
    randn = lambda *s: torch.randn(*s, generator=g)
    d = shape[-1]
    t = {"x": (randn(*shape) * xstd).to(stream), "block": randn(*shape).to(block), "post_weight": (1 + 0.3 * randn(d)).to(weights),
         "pre_weight": (1 + 0.3 * randn(d)).to(weights), "gate": None, "scale": None}
    if gate != "none":
        t["gate"] = (1.5 * randn(*shape[:-1], d if gate == "channel" else 1)).to(block)
    if scale != "none":
        t["scale"] = (0.5 + 0.2 * randn(d) if scale == "channel" else torch.tensor([0.7])).to(weights)
    t = {k: None if v is None else v.to(DEV).requires_grad_() for k, v in t.items()}
    return t, randn(*shape).to(stream).to(DEV), randn(*shape).to(block).to(DEV)


def exact(t, dh, dy, eps=EPS):
    """Outputs and gradients in 64 bits, each with the sum of the magnitudes of its terms."""
    v = {k: None if x is None else x.detach().cpu().double() for k, x in t.items()}
    x, b, wp, wn = v["x"], v["block"], v["post_weight"], v["pre_weight"]
    s = torch.ones(()).double() if v["scale"] is None else v["scale"]
    sig = torch.ones(()).double() if v["gate"] is None else torch.sigmoid(v["gate"])
    mean = lambda a: a.mean(-1, keepdim=True)
    rows = lambda a: a.reshape(-1, a.shape[-1]).sum(0)
    rb = (mean(b * b) + eps).rsqrt()
    nb = b * rb
    part = s * sig * nb * wp
    h = x + part
    rh = (mean(h * h) + eps).rsqrt()
    nh = h * rh
    mh = x.abs() + part.abs()
    out = {"h": (h, mh), "y": (nh * wn, (mh * rh * wn).abs())}
    dh = torch.zeros_like(h) if dh is None else dh.cpu().double()
    dy = torch.zeros_like(h) if dy is None else dy.cpu().double()
    dn, mn = dy * wn, mh * rh
    dx = dh + rh * (dn - nh * mean(dn * nh))
    mx = dh.abs() + rh * (dn.abs() + mn * mean(dn.abs() * mn))
    k = s * sig * wp
    db = rb * (dx * k - nb * mean(dx * k * nb))
    mb = rb * (mx * k.abs() + nb.abs() * mean(mx * (k * nb).abs()))
    q, mq = dx * sig * nb, mx * sig * nb.abs()
    out.update(x=(dx, mx), block=(db, mb), post_weight=(rows(q * s), rows(mq * s.abs())),
               pre_weight=(rows(dy * nh), rows(dy.abs() * mn)))
    if v["gate"] is not None:
        z, mz = dx * s * wp * nb * sig * (1 - sig), mx * (s * wp * nb).abs() * sig
        token = v["gate"].shape != x.shape
        out["gate"] = (z.sum(-1, keepdim=True), mz.sum(-1, keepdim=True)) if token else (z, mz)
    if v["scale"] is not None:
        ds, ms = rows(q * wp), rows(mq * wp.abs())
        out["scale"] = (ds, ms) if v["scale"].numel() == x.shape[-1] else (ds.sum().reshape(v["scale"].shape), ms.sum().reshape(v["scale"].shape))
    return out


def check(t, dh, dy, eps=EPS, layout=lambda a: a):
    args = {k: None if v is None else layout(v) for k, v in t.items()}
    h, y = muon_amd.residual_norm(args["x"], args["block"], args["post_weight"], args["pre_weight"], gate=args["gate"], scale=args["scale"], eps=eps)
    assert h.dtype == t["x"].dtype and y.dtype == t["block"].dtype and h.shape == y.shape == t["x"].shape
    leaves = {k: v for k, v in t.items() if v is not None}
    pairs = [(o, g) for o, g in ((h, dh), (y, dy)) if g is not None]
    grads = dict(zip(leaves, torch.autograd.grad([o for o, _ in pairs], list(leaves.values()), [g for _, g in pairs])))
    want = exact(t, dh, dy, eps)
    rows = t["x"].numel() // t["x"].shape[-1]
    for name, got in {"h": h, "y": y, **grads}.items():
        w, m = want[name]
        factor = 96 if name in ("h", "y") else 192
        if name in ("post_weight", "pre_weight", "scale"):
            factor += rows / 64 + 96
        bound = factor * U * m + UNIT[got.dtype] * w.abs() + 1e-37
        assert got.shape == t[name].shape if name in t else True
        off = (got.detach().cpu().double() - w).abs() - bound
        assert off.max() <= 0, f"{name}: {float(off.max())} over the bound"
    return h, y, grads


WIDTHS = [1, 7, 8, 64, 100, 511, 512, 513, 768, 1024, 1025, 1600, 2048, 2500, 4000, 4096, 4104, 5120, 6000, 7168, 8192, 9001, 16384]


@gpu
@pytest.mark.parametrize("kinds", [(BF16, BF16, BF16), (F32, BF16, F32), (F32, F32, F32), (F32, F32, BF16)], ids=["bf16", "mixed", "fp32", "fp32-bf16"])
@pytest.mark.parametrize("width", WIDTHS)
def test_widths(width, kinds):
    for gate, scale, rows in (("channel", "channel", 5), ("token", "one", 3), ("none", "none", 1)):
        check(*make((rows, width), *kinds, gate=gate, scale=scale, seed=width))


@gpu
@pytest.mark.parametrize("rows", [1, 2, 255, 1025, 4099])
@pytest.mark.parametrize("width", [96, 776, 1600])
def test_rows(rows, width):
    check(*make((rows, width), F32, BF16, F32, gate="token", scale="channel", seed=rows))
    check(*make((rows, width), BF16, BF16, F32, gate="channel", scale="one", seed=rows))


@gpu
def test_more_dimensions_and_other_strides():
    check(*make((3, 5, 7, 40)))
    # rows of a wider tensor, an odd distance apart; a transposed tensor; a broadcast one
    for width, gap in ((768, 5), (100, 3)):
        layout = lambda a: torch.cat([a, a.new_zeros(*a.shape[:-1], gap)], -1)[..., 1 - 1:a.shape[-1]] if a.ndim > 1 else a
        check(*make((9, width)), layout=layout)
        check(*make((9, width)), layout=lambda a: a.t().contiguous().t() if a.ndim > 1 else a)
    t, dh, dy = make((4, 6, 64))
    one = torch.randn(64, device=DEV, dtype=BF16)
    t["block"] = one.expand(4, 6, 64).detach().requires_grad_()
    check(t, dh, dy[..., :1].expand(4, 6, 64))


@gpu
@pytest.mark.parametrize("offset", [1, 2, 3])
@pytest.mark.parametrize("kinds", [(BF16, BF16), (F32, F32)])
def test_any_address(kinds, offset):
    def layout(a):
        buf = torch.zeros(a.numel() + 8, dtype=a.dtype, device=DEV)
        buf[offset:offset + a.numel()] = a.reshape(-1)
        return buf[offset:offset + a.numel()].view(a.shape)

    for width in (72, 1001):
        check(*make((17, width), *kinds, kinds[0], seed=offset), layout=layout)


@gpu
def test_one_gradient_missing_and_inputs_without():
    t, dh, dy = make((33, 200), F32, BF16, F32)
    check(t, dh, None)
    check(t, None, dy)
    for some in (["x"], ["block", "gate"], ["scale"], ["pre_weight"], ["post_weight"]):
        t, dh, dy = make((33, 200), BF16, BF16, F32)
        full = check(t, dh, dy)[2]
        for k, v in t.items():
            v.requires_grad_(k in some)
        h, y = muon_amd.residual_norm(t["x"], t["block"], t["post_weight"], t["pre_weight"], gate=t["gate"], scale=t["scale"], eps=EPS)
        for k, g in zip(some, torch.autograd.grad((h, y), [t[k] for k in some], (dh, dy))):
            assert torch.equal(g, full[k])
    with torch.no_grad():
        h2, y2 = muon_amd.residual_norm(t["x"], t["block"], t["post_weight"], t["pre_weight"], gate=t["gate"], scale=t["scale"], eps=EPS)
    assert torch.equal(h, h2) and torch.equal(y, y2) and not h2.requires_grad


@gpu
def test_gradient_against_differences():
    t, dh, dy = make((6, 40), F32, F32, F32, seed=3)
    _, _, grads = check(t, dh, dy)

    def value(name, delta):
        v = {k: x.detach().cpu().double() for k, x in t.items()}
        v[name] = v[name] + delta
        norm = lambda a: a * (a.pow(2).mean(-1, keepdim=True) + EPS).rsqrt()
        h = v["x"] + v["scale"] * torch.sigmoid(v["gate"]) * norm(v["block"]) * v["post_weight"]
        return float((h * dh.cpu()).sum() + (norm(h) * v["pre_weight"] * dy.cpu()).sum())

    g = torch.Generator().manual_seed(9)
    for name in t:
        d = torch.randn(t[name].shape, generator=g).double()
        step = 1e-4
        slope = (value(name, step * d) - value(name, -step * d)) / (2 * step)
        got = float((grads[name].cpu().double() * d).sum())
        # the difference's own error is of the order step^2 times a third derivative of order 10; the gradient is fp32
        assert abs(got - slope) <= 1e-5 * (1 + float((grads[name].cpu().double() * d).abs().sum()))


@gpu
def test_extremes():
    # rows of zeros, huge and tiny rows, saturated gates
    t, dh, dy = make((8, 96), F32, F32, F32)
    with torch.no_grad():
        t["block"][0] = 0
        t["x"][1] = 0
        t["block"][1] = 0
        t["block"][2] *= 1e15
        t["x"][3] *= 1e15
        t["block"][4] *= 1e-15
        t["gate"][5] = 300
        t["gate"][6] = -300
    check(t, dh, dy)
    t, dh, dy = make((4, 96), F32, F32, F32)
    with torch.no_grad():
        t["block"][1, 5] = float("nan")
        t["x"][2, 7] = float("inf")
    h, y = muon_amd.residual_norm(t["x"], t["block"], t["post_weight"], t["pre_weight"], gate=t["gate"], scale=t["scale"])
    assert torch.isnan(h[1]).all() and torch.isnan(y[1]).all() and torch.isinf(h[2, 7]) and torch.isnan(y[2, 7])
    assert torch.isfinite(h[[0, 3]]).all() and torch.isfinite(y[[0, 3]]).all()      # rows do not touch each other


@gpu
def test_empty():
    for shape in ((0, 64), (5, 0)):
        t, dh, dy = make(shape)
        h, y = muon_amd.residual_norm(t["x"], t["block"], t["post_weight"], t["pre_weight"], gate=t["gate"], scale=t["scale"])
        assert h.shape == y.shape == shape
        for k, g in zip(t, torch.autograd.grad((h, y), list(t.values()), (dh, dy))):
            assert g.shape == t[k].shape and not g.any()


@gpu
def test_repeats_and_streams():
    t, dh, dy = make((3000, 1024), BF16, BF16, F32)
    first = check(t, dh, dy)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = check(t, dh, dy)
    torch.cuda.synchronize()
    assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])
    for k in first[2]:
        assert torch.equal(first[2][k], again[2][k])


@gpu
def test_refusals_on_the_device():
    z = lambda *s, dtype=BF16: torch.zeros(*s, dtype=dtype, device=DEV)
    call = muon_amd.residual_norm
    with pytest.raises(ValueError):
        call(z(2, 8), z(2, 9), z(8), z(8))
    with pytest.raises(ValueError):
        call(z(2, 8), z(2, 8), z(7), z(8))
    with pytest.raises(ValueError):
        call(z(2, 8), z(2, 8), z(8), z(8), scale=z(2))
    with pytest.raises(ValueError):
        call(z(2, 8), z(2, 8), z(8), z(8), gate=z(8))
    with pytest.raises(ValueError):
        call(z(2, 8), z(2, 8), z(8), z(8), eps=-1.0)
    with pytest.raises(ValueError):
        call(z(1, 16385), z(1, 16385), z(16385), z(16385))
    with pytest.raises(TypeError):
        call(z(2, 8), z(2, 8, dtype=F32), z(8), z(8))
    with pytest.raises(TypeError):
        call(z(2, 8), z(2, 8), z(8), z(8, dtype=F32))
    with pytest.raises(TypeError):
        call(z(2, 8), z(2, 8), z(8), z(8), gate=z(2, 8, dtype=F32))
    with pytest.raises(TypeError):
        call(z(2, 8, dtype=torch.float16), z(2, 8), z(8), z(8))
    with pytest.raises(muon_amd.MuonAmdError):
        call(z(2, 8), z(2, 8), z(8), z(8), scale=torch.zeros(8, dtype=BF16))


def test_refusals():
    import ctypes

    from muon_amd import _lib
    z = torch.zeros(2, 8)
    with pytest.raises(muon_amd.MuonAmdError):
        muon_amd.residual_norm(z, z, z[0], z[0])                  # no CPU implementation
    lib = _lib.load()
    assert lib.muon_amd_residual_norm(None, None) == -1 and lib.muon_amd_residual_norm_backward(None, None) == -1
    good = dict(x=4096, b=4096, post_weight=4096, pre_weight=4096, h=4096, y=4096, rows=1, ld_x=8, ld_b=8, width=8, eps=1e-6)
    for bad in (dict(rows=0), dict(width=0), dict(width=20000), dict(x=None), dict(y=None), dict(stream_dtype=1), dict(weight_dtype=7), dict(eps=-1.0)):
        assert lib.muon_amd_residual_norm(ctypes.byref(_lib.ResidualNormArgs(**{**good, **bad})), None) == -1
    # backward without the factors of forward, without a gradient, without a workspace for the sums
    for bad in (dict(), dict(rstd=4096), dict(rstd=4096, dy=4096, dpre_weight=4096)):
        assert lib.muon_amd_residual_norm_backward(ctypes.byref(_lib.ResidualNormArgs(**{**good, **bad})), None) == -1
    assert lib.muon_amd_residual_norm_partials(0, 8) == 0 and lib.muon_amd_residual_norm_partials(100, 8) > 0


@gpu
def test_no_second_derivatives():
    t, dh, dy = make((4, 16), F32, F32, F32)
    h, y = muon_amd.residual_norm(t["x"], t["block"], t["post_weight"], t["pre_weight"], gate=t["gate"], scale=t["scale"])
    g, = torch.autograd.grad((h.sum() + y.sum()), t["x"], create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(g.sum(), t["x"])


@gpu
def test_offsets_beyond_32_bits():
    """More than 2^31 elements in rows a distance apart that passes 2^32 elements over the tensor: the last rows are those
    of a small call, bit for bit."""
    rows, width = 2 ** 31 // 8192 + 7, 8192
    wide = torch.zeros(rows, 2 * width + 8, dtype=BF16, device=DEV)
    x = wide[:, :width]
    t, dh, dy = make((5, width), BF16, BF16, BF16, gate="token", scale="channel")
    x[-5:] = t["x"].detach()
    block, gate = torch.zeros(rows, width, dtype=BF16, device=DEV), torch.zeros(rows, 1, dtype=BF16, device=DEV)
    block[-5:], gate[-5:] = t["block"].detach(), t["gate"].detach()
    gh, gy = torch.zeros_like(block), torch.zeros_like(block)
    gh[-5:], gy[-5:] = dh, dy
    args = [v.requires_grad_() for v in (x, block, gate)]
    small = muon_amd.residual_norm(t["x"], t["block"], t["post_weight"], t["pre_weight"], gate=t["gate"], scale=t["scale"])
    big = muon_amd.residual_norm(args[0], args[1], t["post_weight"], t["pre_weight"], gate=args[2], scale=t["scale"])
    for a, b in zip(small, big):
        assert torch.equal(a, b[-5:]) and not b[:4].any()
    for a, b in zip(torch.autograd.grad(small, [t["x"], t["block"], t["gate"]], (dh, dy)), torch.autograd.grad(big, args, (gh, gy))):
        assert torch.equal(a, b[-5:])
