"""What a language model in training is scored with, and how a balanced mixture of experts routes, as cases that can be
timed: the cross entropy of a linear head over a large vocabulary without its logits, distillation from a teacher's top
logits, and the choice of experts by biased scores within groups of experts.  Each case runs either the framework's
kernels (`own` is true) or the same formulas in elementary torch operations.

A case is a dict of plain values; `kind` says which operator it goes through:

  head     `tokens` hidden states of `width` channels against a `vocab` x `width` matrix, both bf16: every token's loss and
           logsumexp, a share `ignored` of the tokens being padding; `backward`: the mean loss of the others, and the gradients of
           the hidden states and of the matrix, from the loss and from the logsumexps (a z-loss)
  distill  `tokens` rows of `vocab` logits of a student against the `top` largest logits of a teacher and their indices
           (some rows padding, some choices absent), at a temperature: the loss and the gradient of the student's logits
  route    top-`k` of `experts` for `tokens` tokens by score (softmax or sigmoid of the logits) plus a bias for each expert
           (`biased`), among the best `kept` of `groups` groups: indices, weights, tokens per expert, balance loss
           and z-loss, and the gradient of the logits; `masked`: some tokens are padding
"""
import torch

own = False

DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16}
IGNORE = -100
Z_LOSS, BALANCE = 1e-3, 1e-2     # weights of the auxiliary losses in the objective


def listed():
    def head(name, tokens, vocab, width, ignored=0.0, backward=True):
        return dict(name=name, kind="head", tokens=tokens, vocab=vocab, width=width, ignored=ignored, backward=backward)

    def distill(name, tokens, vocab, top, dtype, temperature):
        return dict(name=name, kind="distill", tokens=tokens, vocab=vocab, top=top, dtype=dtype, temperature=temperature)

    def route(name, tokens, experts, k, scores, groups, kept, dtype, biased=True, masked=False):
        return dict(name=name, kind="route", tokens=tokens, experts=experts, k=k, scores=scores, groups=groups, kept=kept, dtype=dtype,
                    biased=biased, masked=masked)

    return [
        # one more token of a sequence is scored: the matrix is read once
        head("head-1x32000x2048-forward", 1, 32000, 2048, backward=False),
        # a short sequence is evaluated with the vocabulary of GPT-2-small
        head("head-64x50257x768-forward", 64, 50257, 768, backward=False),
        # a training micro-batch, vocabulary of 32000
        head("head-4096x32000x2048", 4096, 32000, 2048),
        # ragged: tokens and vocabulary off every power of two, 25 heads of 64, a third of the tokens ignored (prompts)
        head("head-5003x50257x1600-ignored", 5003, 50257, 1600, ignored=0.33),
        # a micro-batch with the vocabulary and width of Llama-3-8B: the largest
        head("head-8192x128256x4096", 8192, 128256, 4096),
        # a few tokens, logits in fp32, eight choices of the teacher
        distill("distill-33x50257-top8-fp32", 33, 50257, 8, "fp32", 1.0),
        # a micro-batch, softened
        distill("distill-4096x32000-top64", 4096, 32000, 64, "bf16", 2.0),
        # the same with a large vocabulary, as many tokens as a step of it holds
        distill("distill-8192x128256-top32", 8192, 128256, 32, "bf16", 1.0),
        # a short batch over few experts, logits in fp32
        route("route-64x16-top2-of-4-groups", 64, 16, 2, "sigmoid", 4, 2, "fp32"),
        # softmax scores, groups of 20 experts, some tokens padding
        route("route-30011x160-top6-softmax", 30011, 160, 6, "softmax", 8, 3, "fp32", masked=True),
        # a long batch over many experts: sigmoid scores, four of eight groups
        route("route-65536x256-top8-sigmoid", 65536, 256, 8, "sigmoid", 8, 4, "bf16"),
    ]


def draw(rng):
    def size(lo, hi):            # spread over the logarithm; odd sizes among them
        return int(round(lo * (hi / lo) ** rng.random()))

    kind = rng.choice(["head", "head", "distill", "route", "route"])
    while True:
        if kind == "head":
            width = size(64, 4096)
            if rng.random() < 0.7:                               # mostly whole heads of 64, sometimes any width
                width = max(64, width // 64 * 64)
            case = dict(kind=kind, tokens=size(1, 8192), vocab=size(1000, 130000), width=width,
                        ignored=rng.choice([0.0, 0.0, 0.1, 0.33, 0.8]), backward=rng.random() < 0.7)
        elif kind == "distill":
            case = dict(kind=kind, tokens=size(1, 8192), vocab=size(1000, 130000), top=size(1, 128),
                        dtype=rng.choice(["fp32", "bf16", "bf16"]), temperature=rng.choice([1.0, 1.0, 0.7, 2.0, 4.0]))
        else:
            groups = rng.choice([1, 1, 2, 4, 8, 16])
            each = size(2, 512 // groups)
            kept = rng.randint(1, groups)
            case = dict(kind=kind, tokens=size(1, 131072), experts=groups * each, k=min(kept * each, rng.choice([1, 2, 4, 6, 8])),
                        scores=rng.choice(["softmax", "sigmoid"]), groups=groups, kept=kept, dtype=rng.choice(["fp32", "bf16"]),
                        biased=rng.random() < 0.8, masked=rng.random() < 0.5)
            if case["scores"] == "softmax" and groups == kept and not case["biased"]:
                continue                                         # (the plain choice by softmax is not what is measured here)
        w = work(case)
        if w["bytes"] <= 6.3e9 and w["flops"] <= 2.5e13:
            return case


# ---- the tensors of a case ---------------------------------------------------------------------------------
def prepare(case, seed):
    """The tensors a user's program has in hand, from the seed alone."""
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)

    def normal(*shape, std=1.0, dtype=torch.float32):
        return torch.empty(*shape, dtype=dtype, device="cuda").normal_(0.0, std, generator=gen)

    def uniform(*shape):
        return torch.rand(*shape, device="cuda", generator=gen)

    n = case["tokens"]
    if case["kind"] == "head":
        v, d = case["vocab"], case["width"]
        weight = normal(v, d, std=2.0 / d ** 0.5, dtype=torch.bfloat16)          # logits of a spread of 2
        target = torch.randint(v, (n,), device="cuda", generator=gen)
        hidden = (normal(n, d) + 1.5 * weight[target].float()).bfloat16()        # the target's is 6 above their mean
        if case["ignored"]:
            target[uniform(n) < case["ignored"]] = IGNORE
        s = {"kind": "head", "backward": case["backward"], "hidden": hidden, "weight": weight, "target": target}
        if case["backward"]:
            hidden.requires_grad_()
            weight.requires_grad_()
            s["dloss"] = torch.ones((), device="cuda")
            s["dlse"] = 2 * Z_LOSS / n * (9.0 + normal(n))       # of a z-loss: in proportion to the logsumexp
        return s
    if case["kind"] == "distill":
        v, k = case["vocab"], case["top"]
        logits = normal(n, v, std=2.0, dtype=DTYPES[case["dtype"]])
        values, indices = [], []
        for rows in logits.split(1024):                          # the teacher's logits are near the student's
            a, b = (rows.float() + normal(*rows.shape)).topk(k)
            values.append(a.to(rows.dtype))
            indices.append(b.int())
        values, indices = torch.cat(values), torch.cat(indices)
        indices[uniform(n, k) < 0.02] = -1                       # a list may be shorter than the others
        indices[uniform(n) < 0.05] = -1                          # padding
        return {"kind": "distill", "temperature": case["temperature"], "logits": logits.requires_grad_(), "values": values,
                "indices": indices, "dloss": torch.ones((), device="cuda")}
    e, k = case["experts"], case["k"]
    s = {"kind": "route", "k": k, "scores": case["scores"], "groups": case["groups"], "kept": case["kept"], "mask": None, "bias": None,
         "logits": normal(n, e, std=1.5, dtype=DTYPES[case["dtype"]]).requires_grad_(), "dweights": normal(n, k, std=1e-2),
         "dbalance": torch.full((), BALANCE, device="cuda"), "dz": torch.full((), Z_LOSS, device="cuda")}
    if case["biased"]:
        s["bias"] = normal(e, std=0.05 if case["scores"] == "sigmoid" else 0.2 / e)
    if case["masked"]:
        s["mask"] = uniform(n) < 0.9
    return s


# ---- one pass ------------------------------------------------------------------------------------------------
def run(state):
    return {"head": _head, "distill": _distill, "route": _route}[state["kind"]](state)


def _head(s):
    h, w, target = s["hidden"], s["weight"], s["target"]
    if own:
        import muon_amd
        out = muon_amd.linear_cross_entropy(h, w, target, ignore_index=IGNORE, reduction="mean" if s["backward"] else "none")
        if not s["backward"]:
            return {"loss": out.loss, "lse": out.lse}
        dh, dw = torch.autograd.grad((out.loss, out.lse), (h, w), (s["dloss"], s["dlse"]))
        return {"loss": out.loss.detach(), "lse": out.lse.detach(), "dhidden": dh, "dweight": dw}
    h, w = h.detach().float(), w.detach().float()
    on = target != IGNORE
    at = torch.where(on, target, 0)[:, None]
    logits = h @ w.t()
    top = logits.amax(1, keepdim=True)
    lse = top + (logits - top).exp().sum(1, keepdim=True).log()
    count = on.sum().clamp(min=1)
    loss = torch.where(on, (lse - logits.gather(1, at))[:, 0], 0.0)
    out = {"loss": loss, "lse": torch.where(on, lse[:, 0], 0.0)}
    if s["backward"]:
        out["loss"] = loss.sum() / count
        each = torch.where(on, s["dloss"] / count, 0.0)[:, None]                 # of each token's loss
        d = (logits - lse).exp_() * (each + torch.where(on, s["dlse"], 0.0)[:, None])
        d.scatter_add_(1, at, -each)
        out.update(dhidden=(d @ w).bfloat16(), dweight=(d.t() @ h).bfloat16())
    return out


def _distill(s):
    x, temperature = s["logits"], s["temperature"]
    if own:
        import muon_amd
        loss = muon_amd.distill_topk(x, s["values"], s["indices"], temperature=temperature)
        grad, = torch.autograd.grad(loss, x, s["dloss"])
        return {"loss": loss.detach(), "grad": grad}
    there = s["indices"] >= 0
    at = torch.where(there, s["indices"], 0).long()
    on = there.any(1, keepdim=True)
    count = on.sum().clamp(min=1)
    y = x.detach().float() / temperature
    top = y.amax(1, keepdim=True)
    lse = top + (y - top).exp().sum(1, keepdim=True).log()
    t = torch.where(there, s["values"].float() / temperature, -torch.inf)
    t = torch.where(on, t, 0.0)
    q = torch.log_softmax(t, 1)
    q, log_q = torch.where(there, q.exp(), 0.0), torch.where(there, q, 0.0)
    loss = temperature ** 2 * (q * (log_q - (y.gather(1, at) - lse))).sum() / count
    d = (y - lse).exp_() * on
    d.scatter_add_(1, at, -q)
    return {"loss": loss, "grad": (d * (s["dloss"] * temperature / count)).to(x.dtype)}


def _plain_route(x, k, scores, bias, groups, kept, mask):
    """-> scores, indices, whether each token takes part, and the share of each expert in its token's scores."""
    n, e = x.shape
    x = x.float()
    on = torch.ones(n, 1, dtype=torch.bool, device=x.device) if mask is None else mask[:, None]
    y = x.detach().double()                                      # what is chosen by: values next to each other
    c = torch.sigmoid(y) if scores == "sigmoid" else torch.softmax(y, 1)
    if bias is not None:
        c = c + bias.double()
    if kept < groups:
        best = c.view(n, groups, -1).topk(min(2, e // groups), 2)[0].sum(2)
        order = torch.sort(best, dim=1, descending=True, stable=True)[1][:, :kept]
        inside = torch.zeros(n, groups, dtype=torch.bool, device=x.device).scatter_(1, order, True)
        c = torch.where(inside.repeat_interleave(e // groups, 1), c, -torch.inf)
    at = torch.sort(c, dim=1, descending=True, stable=True)[1][:, :k]
    s = torch.sigmoid(x) if scores == "sigmoid" else torch.softmax(x, 1)
    return s, at, on, s / s.sum(1, keepdim=True)


def _route(s):
    x, k, mask = s["logits"], s["k"], s["mask"]
    if own:
        import muon_amd
        weights, indices, counts, balance, z = muon_amd.route_topk(x, k, mask=mask, scores=s["scores"], bias=s["bias"], groups=s["groups"],
                                                                   groups_kept=s["kept"])
    else:
        n, e = x.shape
        score, at, on, share = _plain_route(x, k, s["scores"], s["bias"], s["groups"], s["kept"], mask)
        count = on.sum().clamp(min=1)
        chosen = score.gather(1, at).double() * on               # (of the weights' gradients, differences remain: of one choice, nothing)
        weights = (chosen / chosen.sum(1, keepdim=True).clamp(min=1e-30)).float()
        counts = torch.zeros(e, dtype=torch.int64, device=x.device).scatter_add_(0, at.reshape(-1), on.long().expand(n, k).reshape(-1)).int()
        balance = e * ((counts / (count * k)).float() * ((share * on).sum(0) / count)).sum()
        z = (x.float().logsumexp(1) * on[:, 0]).square().sum() / count
        indices = torch.where(on, at, -1).int()
    grad, = torch.autograd.grad((weights, balance, z), x, (s["dweights"], s["dbalance"], s["dz"]))
    return {"weights": weights.detach(), "indices": indices, "counts": counts, "balance": balance.detach(), "z": z.detach(), "grad": grad}


# ---- the definitions in 64 bits --------------------------------------------------------------------------------
def _exact_head(case, seed):
    s = prepare(case, seed)
    h, w, t = s["hidden"].detach().double(), s["weight"].detach().double(), s["target"]
    n = len(h)
    rows = torch.nonzero(t != IGNORE)[:, 0].tolist()
    count = max(len(rows), 1)
    lse = torch.zeros(n, dtype=torch.float64, device="cuda")
    loss = torch.zeros_like(lse)
    dh, dw = torch.zeros_like(h), torch.zeros_like(w)
    for begin in range(0, len(rows), 1024):
        i = torch.tensor(rows[begin:begin + 1024], device="cuda")
        here, cols = torch.arange(len(i), device="cuda"), t[i]
        x = h[i].matmul(w.t())
        lse[i] = torch.logsumexp(x, dim=1)
        loss[i] = lse[i] - x[here, cols]
        if case["backward"]:
            g = s["dloss"].double() / count
            x.sub_(lse[i][:, None]).exp_().mul_((g + s["dlse"][i].double())[:, None])
            x[here, cols] -= g
            dh[i] = x.matmul(w)
            dw += x.t().matmul(h[i])
    out = {"loss": loss.sum() / count if case["backward"] else loss, "lse": lse}
    if case["backward"]:
        out.update(dhidden=dh, dweight=dw)
    return out


def _exact_distill(case, seed):
    s = prepare(case, seed)
    temperature, index = case["temperature"], s["indices"].long()
    active = (index >= 0).any(1)
    count = max(int(active.sum()), 1)
    x = s["logits"].detach()
    total, grad = 0.0, torch.zeros(x.shape, dtype=torch.float64, device="cuda")
    for begin in range(0, len(x), 1024):
        part = slice(begin, begin + 1024)
        use = active[part]
        y = x[part][use].double() / temperature
        i, v = index[part][use], s["values"][part][use].double() / temperature
        v = v.masked_fill(i < 0, -float("inf"))
        q = (v - v.amax(1, keepdim=True)).exp()
        q = q / q.sum(1, keepdim=True)
        log_p = y - torch.logsumexp(y, 1, keepdim=True)
        i = i.clamp(min=0)
        terms = torch.where(q > 0, q * (q.log() - log_p.gather(1, i)), 0.0)
        total = total + terms.sum()
        g = log_p.exp()
        g.scatter_add_(1, i, -q)
        grad[begin:begin + len(use)][use] = g * (temperature * s["dloss"].double() / count)
    return {"loss": torch.as_tensor(total, device="cuda") * temperature ** 2 / count, "grad": grad}


def _exact_route(case, seed):
    s = prepare(case, seed)
    x, k, e, groups, kept = s["logits"].detach().double(), case["k"], case["experts"], case["groups"], case["kept"]
    n, sigmoid = len(x), case["scores"] == "sigmoid"
    on = torch.ones(n, dtype=torch.float64, device="cuda") if s["mask"] is None else s["mask"].double()
    count = max(float(on.sum()), 1.0)
    top = x.amax(1, keepdim=True)
    total = (x - top).exp().sum(1, keepdim=True)
    p = (x - top).exp() / total
    lse = (top + total.log())[:, 0] * on
    score = 1 / (1 + (-x).exp()) if sigmoid else p
    by = score if s["bias"] is None else score + s["bias"].double()
    if kept < groups:
        ranked = torch.sort(by.view(n, groups, e // groups), dim=2, descending=True)[0][:, :, :2].sum(2)
        place = torch.argsort(torch.argsort(-ranked, dim=1, stable=True), dim=1, stable=True)     # of each group in the order
        by = by.view(n, groups, -1).masked_fill((place >= kept)[:, :, None], -float("inf")).view(n, e)
    at = torch.argsort(-by, dim=1, stable=True)[:, :k]
    counts = torch.bincount(at[on > 0].reshape(-1), minlength=e)
    chosen = score.gather(1, at)
    w = chosen / chosen.sum(1, keepdim=True) * on[:, None]
    norm = score.sum(1, keepdim=True)
    share = score / norm
    load = counts.double() / (count * k)
    balance = e * (load * (share * on[:, None]).sum(0) / count).sum()
    u = (BALANCE * e * load / count)[None, :] * on[:, None]
    dscore = (u - (share * u).sum(1, keepdim=True)) / norm
    dw = s["dweights"].double() * on[:, None]
    dscore.scatter_add_(1, at, (dw - (dw * w).sum(1, keepdim=True)) / chosen.sum(1, keepdim=True))
    grad = score * (1 - score) * dscore if sigmoid else p * (dscore - (p * dscore).sum(1, keepdim=True))
    grad = grad + (Z_LOSS * 2 / count * lse)[:, None] * p
    return {"weights": w, "indices": torch.where(on[:, None] > 0, at, -1).int(), "counts": counts.int(), "balance": balance,
            "z": lse.pow(2).sum() / count, "grad": grad}


def exact(case, seed):
    return {"head": _exact_head, "distill": _exact_distill, "route": _exact_route}[case["kind"]](case, seed)


# ---- what a pass cannot do without -----------------------------------------------------------------------------
def work(case):
    n = case["tokens"]
    if case["kind"] == "head":
        v, d = case["vocab"], case["width"]
        taking = n * (1 - case["ignored"])                       # tokens that take part: those have logits
        read, products = 2 * d * (taking + v) + 12 * n, 1
        if case["backward"]:                                     # the gradients of both, and the two products behind them
            read, products = read + 2 * d * (n + v) + 4 * n, 3
        return {"bytes": int(read), "flops": int(2 * taking * v * d * products)}
    e = 4 if case["dtype"] == "fp32" else 2
    if case["kind"] == "distill":                                # logits in, gradient out, the teacher's
        return {"bytes": n * (2 * case["vocab"] * e + case["top"] * (e + 4)), "flops": n * case["vocab"] * 8}
    m, k = case["experts"], case["k"]
    return {"bytes": n * (2 * m * e + 12 * k + (1 if case["masked"] else 0)) + 8 * m, "flops": n * m * (12 + 2 * k)}
