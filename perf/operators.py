"""The operators of a training step around the matrices that Muon updates, as cases that can be timed:
the AdamW step of everything that is not such a matrix, clipping by the norm of all gradients, the norms
on both sides of a transformer block with its gate and residual scale, and a router with its balance
loss.  Each case runs either the framework's kernels (`own` is true) or the same formulas in elementary
torch operations.

A case is a dict of plain values; `kind` says which operator it goes through:

  adamw     AdamW over one matrix of `rows` x `width` and `vectors` vectors of `width` elements and less, states in
            `bits` bits; `clip`: the gradients are scaled by the coefficient of their joint norm on the way.
            States of 8 bits are returned as the values they stand for
  clip      the gradients of `layers` blocks of `width` (key/value width `kv`, feed-forward width `ff`) and of
            `vectors` vectors, scaled in place to a joint norm of at most a given one
  residual  the residual step between two blocks over `tokens` rows of `width`:
            h = x + scale * sigmoid(gate) * norm(b) * post_weight,  y = norm(h) * pre_weight
            with the gate per channel, per token or absent, and (`backward`) the gradients of all inputs
  route     top-`k` of `experts` for `tokens` tokens: indices, weights, tokens per expert, balance loss and
            z-loss, and the gradient of the logits; `masked`: some tokens are padding

Tensors of an optimizer are views into one flat buffer per role, as programs keep them that reduce or save
them in one piece; the plain forms work on the whole buffers (what lies between two tensors is zero).
"""
import torch

own = False

DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16}
LR, BETAS, EPS, WEIGHT_DECAY = 3e-4, (0.9, 0.95), 1e-8, 0.01
FIRST_STEP = 100                 # steps that the optimizer's state has behind it
GRAD_STD, PARAM_STD = 1e-3, 0.02
NORM_EPS = 1e-6
BALANCE, Z_LOSS = 1e-2, 1e-3     # weights of the two losses in the objective
BLOCK = 128                      # elements that share the exponent of an 8-bit state, and the unit of the flat buffers


def listed():
    def adamw(name, rows, width, vectors, dtype, bits, clip=False):
        return dict(name=name, kind="adamw", rows=rows, width=width, vectors=vectors, dtype=dtype, bits=bits, clip=clip)

    def residual(name, tokens, width, stream, dtype, gate, scaled=True, backward=True):
        return dict(name=name, kind="residual", tokens=tokens, width=width, stream=stream, dtype=dtype, gate=gate,
                    scaled=scaled, backward=backward)

    return [
        # the smallest call: the norm weights and biases of GPT-2-small, states in 32 bits
        adamw("adamw32-norms-49x768", 0, 768, 49, "fp32", 32),
        # the vocabulary matrix of GPT-2-small and its norm weights kept in bf16, states in 8 bits
        adamw("adamw8-50257x768-bf16", 50257, 768, 25, "bf16", 8),
        # a vocabulary of 32000 in bf16 with states in 32 bits, the gradients clipped on the way
        adamw("adamw32-clip-32000x2048-bf16", 32000, 2048, 25, "bf16", 32, clip=True),
        # one vocabulary matrix of Llama-3-8B and its 65 norm weights, states in 8 bits: the largest
        adamw("adamw8-128256x4096", 128256, 4096, 65, "fp32", 8),
        # a few vectors: the latency of clipping
        dict(name="clip-49x768", kind="clip", layers=0, width=768, kv=768, ff=0, vectors=49, dtype="fp32"),
        # every gradient of a bf16 model with grouped key/value heads and a feed-forward of 21.5 tiles
        dict(name="clip-decoder-2048-bf16", kind="clip", layers=12, width=2048, kv=512, ff=5504, vectors=25, dtype="bf16"),
        # a single sequence's few tokens, forward only: what a step costs that evaluates
        residual("residual-33x768-forward", 33, 768, "bf16", "bf16", "channel", backward=False),
        # a micro-batch of a medium model, one gate for each token
        residual("residual-8192x2048-token", 8192, 2048, "bf16", "bf16", "token"),
        # ragged: a number of tokens off every power of two, 25 heads of 64, a residual stream in fp32
        residual("residual-5003x1600-fp32", 5003, 1600, "fp32", "bf16", "channel"),
        # a batch of a large model's tokens, gate for each channel
        residual("residual-16384x4096", 16384, 4096, "bf16", "bf16", "channel"),
        # a short batch over few experts, logits in fp32
        dict(name="route-1024x8-top2", kind="route", tokens=1024, experts=8, k=2, dtype="fp32", masked=False),
        # a long batch over many experts, some tokens padding
        dict(name="route-65536x256-top8", kind="route", tokens=65536, experts=256, k=8, dtype="bf16", masked=True),
    ]


def draw(rng):
    def size(lo, hi):            # spread over the logarithm; odd sizes among them
        return int(round(lo * (hi / lo) ** rng.random()))

    kind = rng.choice(["adamw", "adamw", "clip", "residual", "residual", "route"])
    while True:
        if kind == "adamw":
            case = dict(kind=kind, rows=rng.choice([0, size(1, 130000), size(1000, 130000)]), width=size(64, 4096),
                        vectors=size(1, 130), dtype=rng.choice(["fp32", "bf16"]), bits=rng.choice([8, 32]),
                        clip=rng.random() < 0.3)
        elif kind == "clip":
            width = size(64, 4096)
            case = dict(kind=kind, layers=rng.choice([0, size(1, 12)]), width=width, kv=max(1, width // rng.choice([1, 4])),
                        ff=size(width, 4 * width), vectors=size(1, 130), dtype=rng.choice(["fp32", "bf16"]))
        elif kind == "residual":
            dtype = rng.choice(["bf16", "bf16", "fp32"])
            width = size(64, 8192)
            if rng.random() < 0.7:                               # mostly whole heads of 64, sometimes any width
                width = max(64, width // 64 * 64)
            case = dict(kind=kind, tokens=size(1, 32768), width=width, stream="fp32" if rng.random() < 0.3 else dtype,
                        dtype=dtype, gate=rng.choice(["channel", "token", "none"]), scaled=rng.random() < 0.75,
                        backward=rng.random() < 0.75)
        else:
            experts = size(4, 512)
            case = dict(kind=kind, tokens=size(1, 131072), experts=experts, k=min(experts, rng.choice([1, 2, 4, 6, 8])),
                        dtype=rng.choice(["fp32", "bf16"]), masked=rng.random() < 0.5)
        if work(case)["bytes"] <= 1.0e10:                        # well under the largest listed case
            return case


# ---- the tensors of a case -------------------------------------------------------------------------------
def _shapes(case):
    w = case["width"]
    if case["kind"] == "adamw":
        matrices = [(case["rows"], w)] if case["rows"] else []
    else:
        matrices = [(w, w), (case["kv"], w), (case["kv"], w), (w, w), (case["ff"], w), (case["ff"], w), (w, case["ff"])] * case["layers"]
    return matrices + [(w - 37 * j % (w // 2 + 1),) for j in range(case["vectors"])]


def _numel(shape):
    n = 1
    for s in shape:
        n *= s
    return n


def _starts(shapes):
    starts, end = [], 0
    for s in shapes:
        starts.append(end)
        end += -(-_numel(s) // BLOCK) * BLOCK
    return starts, end


def _views(buf, shapes, starts):
    return [buf[o:o + _numel(s)].view(s) for o, s in zip(starts, shapes)]


def _inputs(case, seed):
    """The tensors a user's program has in hand, from the seed alone."""
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    kind, dtype = case["kind"], DTYPES[case["dtype"]]

    def normal(*shape, std=1.0, mean=0.0, dtype=dtype):
        return torch.empty(*shape, dtype=dtype, device="cuda").normal_(mean, std, generator=gen)

    if kind in ("adamw", "clip"):
        shapes = _shapes(case)
        starts, end = _starts(shapes)
        inside = torch.zeros(end, dtype=torch.bool, device="cuda")
        for v in _views(inside, shapes, starts):
            v.fill_(True)

        def flat(std, dtype=dtype):
            return normal(end, std=std, dtype=dtype).mul_(inside)

        s = {"kind": kind, "shapes": shapes, "starts": starts, "grad": flat(GRAD_STD)}
        if kind == "clip":
            s["max_norm"] = 0.5 * GRAD_STD * sum(map(_numel, shapes)) ** 0.5
            return s
        s.update(param=flat(PARAM_STD), bits=case["bits"], step=FIRST_STEP, clip=case["clip"],
                 max_norm=0.5 * GRAD_STD * sum(map(_numel, shapes)) ** 0.5)
        m, v = flat(0.3 * GRAD_STD, torch.float32), flat(GRAD_STD, torch.float32).square_()
        if case["bits"] == 32:
            s.update(m=m, v=v)
            return s
        # where each block of 128 starts within its tensor: the dither of an element goes by its place there
        counts = torch.tensor([-(-_numel(t) // BLOCK) for t in shapes], device="cuda")
        first = torch.tensor([o // BLOCK for o in starts], device="cuda")
        blocks = torch.arange(end // BLOCK, device="cuda")
        s["place"] = ((blocks - first.repeat_interleave(counts)) * BLOCK).to(torch.int32)
        s["mc"], s["me"], s["vc"], s["ve"] = _encode(m, v, s["place"], FIRST_STEP)
        return s
    if kind == "residual":
        t, w, stream = case["tokens"], case["width"], DTYPES[case["stream"]]
        s = {"kind": kind, "backward": case["backward"], "x": normal(t, w, std=2.0, dtype=stream), "b": normal(t, w),
             "post": normal(w, std=0.1, mean=1.0), "pre": normal(w, std=0.1, mean=1.0),
             "gate": {"channel": lambda: normal(t, w), "token": lambda: normal(t, 1), "none": lambda: None}[case["gate"]](),
             "scale": normal(w, std=0.05, mean=0.5) if case["scaled"] else None}
        if case["backward"]:
            s.update(dh=normal(t, w, std=1e-2, dtype=stream), dy=normal(t, w, std=1e-2))
            for name in ("x", "b", "post", "pre", "gate", "scale"):
                if s[name] is not None:
                    s[name].requires_grad_()
        return s
    t, e = case["tokens"], case["experts"]
    s = {"kind": kind, "k": case["k"], "logits": normal(t, e, std=1.5).requires_grad_(),
         "dweights": normal(t, case["k"], std=1e-2, dtype=torch.float32), "mask": None}
    if case["masked"]:
        s["mask"] = torch.rand(t, device="cuda", generator=gen) < 0.9
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    if own and case["kind"] in ("adamw", "clip"):                # parameters, and the optimizer that holds them
        import muon_amd
        shapes, starts = s["shapes"], s["starts"]
        s["params"] = [torch.nn.Parameter(v) for v in _views(s["param"] if "param" in s else torch.zeros_like(s["grad"]), shapes, starts)]
        for p, g in zip(s["params"], _views(s["grad"], shapes, starts)):
            p.grad = g
        if case["kind"] == "adamw":
            opt = s["opt"] = muon_amd.AdamW(s["params"], lr=LR, betas=BETAS, eps=EPS, weight_decay=WEIGHT_DECAY,
                                            state_bits=case["bits"])
            names = ("m", "v") if case["bits"] == 32 else ("mc", "vc")
            for p, o, m, v in zip(s["params"], starts, *(_views(s[n], shapes, starts) for n in names)):
                opt.state[p].update(exp_avg=m, exp_avg_sq=v, step=FIRST_STEP)
                if case["bits"] == 8:
                    b = slice(o // BLOCK, o // BLOCK + -(-p.numel() // BLOCK))
                    opt.state[p].update(exp_avg_exponent=s["me"][b], exp_avg_sq_exponent=s["ve"][b])
            if case["bits"] == 8:
                s["values"] = [torch.zeros_like(s["mc"], dtype=torch.bfloat16) for _ in range(2)]
                s["value_views"] = list(zip(*(_views(v, shapes, starts) for v in s["values"])))
    return s


# ---- one pass ----------------------------------------------------------------------------------------------
def run(state):
    return {"adamw": _adamw, "clip": _clip, "residual": _residual, "route": _route}[state["kind"]](state)


def _plain_coefficient(grad, max_norm):
    norm = grad.float().square().sum().sqrt()
    return norm, (max_norm / (norm + 1e-6)).clamp(max=1.0)


def _wrap(c):                    # as a signed 32-bit factor
    return c - (1 << 32) if c >= 1 << 31 else c


def _mix(step):
    """32 bits that go by the step alone: multiplications by odd numbers and exclusive ors with what is shifted down."""
    x = step * 0x9E3779B9 & 0xFFFFFFFF
    x = (x ^ x >> 16) * 0xC13FA9A9 & 0xFFFFFFFF
    x = (x ^ x >> 15) * 0x91E10DA5 & 0xFFFFFFFF
    return x ^ x >> 16


def _dither(place, step):
    """20 bits for each element and moment, by the element's place in its tensor and the step."""
    h = (place[:, None] + torch.arange(BLOCK, dtype=torch.int32, device=place.device)) * _wrap(0x9E3779B9) + _wrap(_mix(step))
    x = (h ^ (h >> 15 & 0x1FFFF)) & 0xFFFFFF
    return x * 0xC13FA9 >> 12 & 0xFFFFF, x * 0x91E10D >> 12 & 0xFFFFF


def _scaled(x, n):
    """x * 2^n, exactly (torch.ldexp goes through pow, which is a unit off for some n on the GPU)."""
    return x * (n + 127 << 23).view(torch.float32)


def _encode(m, v, place, step):
    """8-bit states: per block of 128 the exponent of the largest magnitude (rounded up where the element's own
    code would pass the largest one), per element three bits of mantissa and four (m: the codes of float8_e4m3fn) or
    five (v, unsigned) of exponent, rounded by a dither; a v above zero never becomes zero."""
    out = []
    for x, top, carry, dither in zip((m, v), (15, 31), (0x1FFFFF, 0xFFFFF), _dither(place, step)):
        x = x.view(-1, BLOCK)
        most = x.abs().amax(1, keepdim=True).view(torch.int32)
        e = (most + carry) >> 23
        code = (_scaled(x.abs(), top - e).view(torch.int32) + dither) >> 20
        code = code | ((x.view(torch.int32) >> 24) & 0x80) if top == 15 else torch.where(x > 0, code.clamp(min=1), code)
        out += [code.to(torch.uint8).view(-1), e.to(torch.uint8).view(-1)]
    return out


def _decode(code, e, top):
    c, e = code.view(-1, BLOCK).to(torch.int32), e.view(-1, 1).to(torch.int32)
    if top == 15:
        x = _scaled(((c & 0x7F) << 20).view(torch.float32), e - top)
        return torch.where(c > 0x7F, -x, x).view(-1)
    return _scaled((c << 20).view(torch.float32), e - top).view(-1)


def _adamw(s):
    if own:
        import muon_amd
        if s["clip"]:
            norm, coefficient = muon_amd.clip_coefficient(s["params"], s["max_norm"])
            s["opt"].step(grad_scale=coefficient)
        else:
            norm = None
            s["opt"].step()
        if s["bits"] == 8:
            s["opt"].state_values(out=s["value_views"])
            return {"param": s["param"], "m": s["values"][0], "v": s["values"][1], "norm": norm}
        return {"param": s["param"], "m": s["m"], "v": s["v"], "norm": norm}
    s["step"] += 1
    step, (b1, b2), norm = s["step"], BETAS, None
    g = s["grad"].float()
    if s["clip"]:
        norm, coefficient = _plain_coefficient(s["grad"], s["max_norm"])
        g = g * coefficient
    m, v = (s["m"], s["v"]) if s["bits"] == 32 else (_decode(s["mc"], s["me"], 15), _decode(s["vc"], s["ve"], 31))
    m.lerp_(g, 1 - b1)
    v.lerp_(g * g, 1 - b2)
    denominator = v.sqrt().mul_((1 - b2 ** step) ** -0.5).add_(EPS)
    s["param"].copy_(s["param"].float().mul_(1 - LR * WEIGHT_DECAY).addcdiv_(m, denominator, value=-LR / (1 - b1 ** step)))
    if s["bits"] == 8:
        s["mc"], s["me"], s["vc"], s["ve"] = _encode(m, v, s["place"], step)
        m, v = _decode(s["mc"], s["me"], 15).bfloat16(), _decode(s["vc"], s["ve"], 31).bfloat16()
    return {"param": s["param"], "m": m, "v": v, "norm": norm}


def _clip(s):
    # the threshold sinks a little from pass to pass, so that there is something to scale in each
    s["max_norm"] *= 0.9999
    if own:
        import muon_amd
        return {"grad": s["grad"], "norm": muon_amd.clip_grad_norm_(s["params"], s["max_norm"])}
    norm, coefficient = _plain_coefficient(s["grad"], s["max_norm"])
    s["grad"].copy_(s["grad"].float() * coefficient)
    return {"grad": s["grad"], "norm": norm}


def _plain_residual(x, b, post, pre, gate, scale):
    def norm(t):
        return t * torch.rsqrt(t.square().mean(-1, keepdim=True) + NORM_EPS)

    u = norm(b.float()) * post.float()
    if gate is not None:
        u = u * torch.sigmoid(gate.float())
    if scale is not None:
        u = u * scale.float()
    h = x.float() + u
    return h.to(x.dtype), (norm(h) * pre.float()).to(b.dtype)


def _residual(s):
    args = s["x"], s["b"], s["post"], s["pre"], s["gate"], s["scale"]
    if own:
        import muon_amd
        h, y = muon_amd.residual_norm(*args[:4], gate=s["gate"], scale=s["scale"], eps=NORM_EPS)
    else:
        h, y = _plain_residual(*args)
    if not s["backward"]:
        return {"h": h, "y": y}
    leaves = [t for t in args if t is not None]
    return {"h": h.detach(), "y": y.detach(), "grads": torch.autograd.grad((h, y), leaves, (s["dh"], s["dy"]))}


def _plain_route(logits, k, mask):
    x = logits.float()
    lse = x.logsumexp(-1)
    p = (x - lse[:, None]).exp()
    at = torch.sort(x.detach(), dim=-1, descending=True, stable=True)[1][:, :k]
    if mask is not None:
        lse, p = lse * mask, p * mask[:, None]
    chosen = p.gather(-1, at)
    weights = chosen / chosen.sum(-1, keepdim=True).clamp(min=1e-30)
    hits = torch.ones_like(at) if mask is None else mask[:, None].expand_as(at).long()
    counts = torch.zeros(x.shape[1], dtype=torch.int64, device=x.device).scatter_add_(0, at.reshape(-1), hits.reshape(-1))
    n = x.shape[0] if mask is None else mask.sum().clamp(min=1)
    balance = x.shape[1] * ((counts / (n * k)).float() * (p.sum(0) / n)).sum()
    if mask is not None:
        at = torch.where(mask[:, None], at, -1)
    return weights, at.to(torch.int32), counts.to(torch.int32), balance, lse.square().sum() / n


def _route(s):
    if own:
        import muon_amd
        weights, indices, counts, balance, z = muon_amd.route_topk(s["logits"], s["k"], mask=s["mask"])
    else:
        weights, indices, counts, balance, z = _plain_route(s["logits"], s["k"], s["mask"])
    losses = torch.full((), BALANCE, device="cuda"), torch.full((), Z_LOSS, device="cuda")
    grad, = torch.autograd.grad((weights, balance, z), s["logits"], (s["dweights"], *losses))
    return {"weights": weights.detach(), "indices": indices, "counts": counts, "balance": balance.detach(), "z": z.detach(), "grad": grad}


# ---- the definitions in 64 bits ------------------------------------------------------------------------------
def _exact_state(x, top, factor, step):
    """x (one tensor's moment) as its 8-bit codes' values: to a multiple of 2^-3 of its own power of two (of the
    lowest one below that), up with the chance that the dither's 20 bits give."""
    n = x.numel()
    pad = torch.zeros(-(-n // BLOCK) * BLOCK - n, dtype=torch.float64, device=x.device)
    blocks = torch.cat([x, pad]).view(-1, BLOCK)
    most = blocks.abs().amax(1, keepdim=True)
    mantissa, exponent = torch.frexp(most)                        # most = mantissa * 2^exponent, mantissa in [1/2, 1)
    exponent = torch.where(mantissa > (14 / 16 if top == 15 else 15 / 16), exponent, exponent - 1)
    own_power = torch.frexp(blocks.abs())[1] - 1
    power = torch.maximum(own_power, exponent - (top - 1))
    step_size = torch.pow(2.0, (power - 3).double())
    i = torch.arange(blocks.numel(), device=x.device, dtype=torch.int64).view(-1, BLOCK)
    h = (i * 0x9E3779B9 + _mix(step)) % (1 << 32)
    u = ((h ^ h >> 15) % (1 << 24) * factor % (1 << 32) >> 12).double() / (1 << 20)
    q = torch.floor(blocks.abs() / step_size + u)
    if top == 31:
        q = torch.where(blocks > 0, q.clamp(min=1), q)
    return torch.where(most > 0, q * step_size * blocks.sign(), 0.0).view(-1)[:n]


def _exact_optimizer(case, seed):
    s = _inputs(case, seed)
    total = s["grad"].double().square().sum().sqrt()
    factor = (s["max_norm"] * (0.9999 if case["kind"] == "clip" else 1.0) / (total + 1e-6)).clamp(max=1.0)
    if case["kind"] == "clip":
        return {"grad": s["grad"].double() * factor, "norm": total}
    t, (b1, b2) = FIRST_STEP + 1, BETAS
    g = s["grad"].double() * (factor if case["clip"] else 1.0)
    if case["bits"] == 32:
        m, v = s["m"].double(), s["v"].double()
    else:
        m, v = _decode(s["mc"], s["me"], 15).double(), _decode(s["vc"], s["ve"], 31).double()
    m = b1 * m + (1 - b1) * g
    v = b2 * v + (1 - b2) * g * g
    update = (m / (1 - b1 ** t)) / ((v / (1 - b2 ** t)).sqrt() + EPS)
    param = s["param"].double() * (1 - LR * WEIGHT_DECAY) - LR * update
    if case["bits"] == 8:
        mq, vq = torch.zeros_like(m), torch.zeros_like(v)
        for o, shape in zip(s["starts"], s["shapes"]):
            at = slice(o, o + _numel(shape))
            mq[at] = _exact_state(m[at], 15, 0xC13FA9, t)
            vq[at] = _exact_state(v[at], 31, 0x91E10D, t)
        m, v = mq, vq
    return {"param": param, "m": m, "v": v, "norm": total if case["clip"] else None}


def _exact_residual(case, seed):
    s = _inputs(case, seed)
    x, b, post, pre, gate, scale = (None if s[n] is None else s[n].detach().double() for n in ("x", "b", "post", "pre", "gate", "scale"))
    rb = 1 / (b.pow(2).mean(-1, keepdim=True) + NORM_EPS).sqrt()
    nb = b * rb
    sig = 1 / (1 + (-gate).exp()) if gate is not None else torch.ones((), dtype=torch.float64, device="cuda")
    lam = scale if scale is not None else torch.ones((), dtype=torch.float64, device="cuda")
    h = x + lam * sig * nb * post
    rh = 1 / (h.pow(2).mean(-1, keepdim=True) + NORM_EPS).sqrt()
    nh = h * rh
    if not case["backward"]:
        return {"h": h, "y": nh * pre}
    dy = s["dy"].double()
    dn = dy * pre
    dx = s["dh"].double() + rh * (dn - nh * (dn * nh).mean(-1, keepdim=True))
    du = dx * lam * sig                                   # gradient of norm(b) * post
    dnb = du * post
    grads = [dx, rb * (dnb - nb * (dnb * nb).mean(-1, keepdim=True)), (du * nb).sum(0), (dy * nh).sum(0)]
    if gate is not None:
        dg = dx * lam * nb * post * sig * (1 - sig)
        grads.append(dg if case["gate"] == "channel" else dg.sum(-1, keepdim=True))
    if scale is not None:
        grads.append((dx * sig * nb * post).sum(0))
    return {"h": h, "y": nh * pre, "grads": grads}


def _exact_route(case, seed):
    s = _inputs(case, seed)
    x, k, e = s["logits"].detach().double(), case["k"], case["experts"]
    on = torch.ones(len(x), dtype=torch.float64, device="cuda") if s["mask"] is None else s["mask"].double()
    n = max(float(on.sum()), 1.0)
    top = x.amax(-1, keepdim=True)
    total = (x - top).exp().sum(-1, keepdim=True)
    lse = (top + total.log())[:, 0] * on
    p = (x - top).exp() / total * on[:, None]
    at = torch.argsort(-x, dim=-1, stable=True)[:, :k]
    counts = torch.bincount(at[on > 0].reshape(-1), minlength=e)
    chosen = p.gather(1, at)
    w = chosen / chosen.sum(-1, keepdim=True).clamp(min=1e-300)
    share = counts.double() / (n * k)
    balance = e * (share * p.sum(0) / n).sum()
    dp = BALANCE * e * share / n
    grad = p * (dp - (p * dp).sum(-1, keepdim=True)) + Z_LOSS * 2 / n * lse[:, None] * p
    dw = s["dweights"].double() * on[:, None]
    grad.scatter_add_(1, at, w * (dw - (w * dw).sum(-1, keepdim=True)))
    return {"weights": w, "indices": torch.where(on[:, None] > 0, at, -1).int(), "counts": counts.int(), "balance": balance,
            "z": lse.pow(2).sum() / n, "grad": grad}


def exact(case, seed):
    return {"adamw": _exact_optimizer, "clip": _exact_optimizer, "residual": _exact_residual, "route": _exact_route}[case["kind"]](case, seed)


# ---- what a pass cannot do without ---------------------------------------------------------------------------
def work(case):
    e = 4 if case["dtype"] == "fp32" else 2
    if case["kind"] in ("adamw", "clip"):
        n = sum(map(_numel, _shapes(case)))
        if case["kind"] == "clip":
            return {"bytes": 2 * e * n, "flops": 3 * n}
        # parameter read and written, gradient read, both states read and written; 8-bit states: codes, a byte for each
        # block, and the values of both in bf16
        states = 16 if case["bits"] == 32 else 4 + 4 / BLOCK + 4
        return {"bytes": n * (3 * e + states), "flops": n * (14 if case["bits"] == 32 else 30)}
    if case["kind"] == "residual":
        t, w, x = case["tokens"], case["width"], 4 if case["stream"] == "fp32" else 2
        gate = {"channel": w * e, "token": e, "none": 0}[case["gate"]]
        vectors = (2 + case["scaled"]) * w * e
        forward = t * (2 * w * x + 2 * w * e + gate) + vectors                   # x, h; b, y; the gate
        backward = t * (2 * w * x + 2 * w * e + gate) + vectors if case["backward"] else 0     # dh, dx; dy, db; the gate's
        return {"bytes": forward + backward, "flops": t * w * (12 + (30 if case["backward"] else 0))}
    t, n, k = case["tokens"], case["experts"], case["k"]
    return {"bytes": t * (2 * n * e + 12 * k + (1 if case["masked"] else 0)) + 4 * n, "flops": t * n * (8 + 2 * k)}
