"""Operators of a transformer's forward and backward pass whose weights the optimizers of this package train, as torch
functions with gradients.

    residual_norm(x, block, post_weight, pre_weight, gate=..., scale=...)  -> h, y
        the norm after a block, its gate and residual scale, the addition to the residual stream, and the norm before
        the next block, in one pass
    route_topk(logits, k)  -> weights, indices, counts, balance_loss, z_loss
        the experts of each token, tokens per expert, and the losses that keep them balanced
"""
from __future__ import annotations

import ctypes
from typing import NamedTuple

import torch

from . import _lib
from .engine import _launch, _stream_ptr, require_gpu_tensor

_DTYPES = {torch.float32: _lib.SRC_F32, torch.bfloat16: _lib.SRC_BF16}


def _dtype(t: torch.Tensor, name: str) -> int:
    try:
        return _DTYPES[t.dtype]
    except KeyError:
        raise TypeError(f"{name} is {t.dtype}: fp32 and bf16 tensors are taken") from None


def _rows(t: torch.Tensor, width: int) -> torch.Tensor:
    """`t` as rows of `width` elements next to each other (any distance between rows): a view where its strides allow
    that, else a copy."""
    t = t.reshape(-1, width)
    return t if width == 1 or t.stride(1) == 1 else t.contiguous()


class _ResidualNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, block, post_weight, pre_weight, gate, scale, eps):
        width, rows = x.size(-1), x.numel() // max(x.size(-1), 1)
        h, y = torch.empty(x.shape, dtype=x.dtype, device=x.device), torch.empty(x.shape, dtype=block.dtype, device=x.device)
        ctx.set_materialize_grads(False)
        ctx.eps = eps
        if rows == 0 or width == 0:
            ctx.save_for_backward(x, block, post_weight, pre_weight, gate, scale, None)
            return h, y
        needed = any(ctx.needs_input_grad)
        rstd = torch.empty(rows, 2, dtype=torch.float32, device=x.device) if needed else None
        a, keep = _residual_args(x, block, post_weight, pre_weight, gate, scale, eps)
        a.h, a.y, a.rstd = h.data_ptr(), y.data_ptr(), rstd.data_ptr() if needed else None
        with torch.cuda.device(x.device):
            _launch("residual_norm", 2 * (h.numel() * h.element_size() + y.numel() * y.element_size()), lambda: _lib.check(
                _lib.load().muon_amd_residual_norm(ctypes.byref(a), _stream_ptr(x.device)), "residual_norm"))
        if needed:
            ctx.save_for_backward(x, block, post_weight, pre_weight, gate, scale, rstd)
        return h, y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dh, dy):
        x, block, post_weight, pre_weight, gate, scale, rstd = ctx.saved_tensors
        inputs = (x, block, post_weight, pre_weight, gate, scale)
        if rstd is None or (dh is None and dy is None):
            return (*(torch.zeros_like(t) if n and t is not None else None for t, n in zip(inputs, ctx.needs_input_grad)), None)
        grads = [torch.empty(t.shape, dtype=t.dtype, device=t.device) if n and t is not None else None
                 for t, n in zip(inputs, ctx.needs_input_grad)]
        a, keep = _residual_args(*inputs, ctx.eps)
        width = a.width
        if dh is not None:
            dh = _rows(dh, width)
            a.dh, a.ld_dh = dh.data_ptr(), dh.stride(0)
        if dy is not None:
            dy = _rows(dy, width)
            a.dy, a.ld_dy = dy.data_ptr(), dy.stride(0)
        a.rstd = rstd.data_ptr()
        a.dx, a.db, a.dpost_weight, a.dpre_weight, a.dgate, a.dscale = (None if g is None else g.data_ptr() for g in grads)
        lib = _lib.load()
        if a.dpost_weight or a.dpre_weight or a.dscale:
            partials = torch.empty(lib.muon_amd_residual_norm_partials(a.rows, width), dtype=torch.float32, device=x.device)
            a.partials = partials.data_ptr()
        with torch.cuda.device(x.device):
            _launch("residual_norm_backward", 3 * x.numel() * (x.element_size() + block.element_size()), lambda: _lib.check(
                lib.muon_amd_residual_norm_backward(ctypes.byref(a), _stream_ptr(x.device)), "residual_norm_backward"))
        return (*grads, None)


def _residual_args(x, block, post_weight, pre_weight, gate, scale, eps):
    """The arguments of both directions, and the tensors behind the addresses in them."""
    width = x.size(-1)
    xr, br = _rows(x, width), _rows(block, width)
    post, pre = post_weight.contiguous(), pre_weight.contiguous()
    a = _lib.ResidualNormArgs(x=xr.data_ptr(), b=br.data_ptr(), post_weight=post.data_ptr(), pre_weight=pre.data_ptr(), rows=xr.size(0),
                              ld_x=xr.stride(0), ld_b=br.stride(0), width=width, stream_dtype=_DTYPES[x.dtype],
                              block_dtype=_DTYPES[block.dtype], weight_dtype=_DTYPES[post.dtype], eps=eps)
    keep = [xr, br, post, pre]
    if gate is not None:
        gr = _rows(gate, gate.size(-1))
        a.gate, a.ld_gate, a.gate_is_token = gr.data_ptr(), gr.stride(0), int(gate.size(-1) != width)
        keep.append(gr)
    if scale is not None:
        sr = scale.contiguous()
        a.scale, a.scale_is_one = sr.data_ptr(), int(sr.numel() != width)
        keep.append(sr)
    return a, keep


def residual_norm(x: torch.Tensor, block: torch.Tensor, post_weight: torch.Tensor, pre_weight: torch.Tensor, *,
                  gate: torch.Tensor | None = None, scale: torch.Tensor | None = None, eps: float = 1e-6):
    """The step between two blocks of a transformer over rows of D channels (the last dimension):

        h = x + scale * sigmoid(gate) * norm(block) * post_weight
        y = norm(h) * pre_weight                          norm(t) = t / sqrt(mean(t^2) + eps)

    x: the residual stream, fp32 or bf16; block: the output of the block that just ran, of x's shape, bf16 or x's type.
    gate: logits in block's type, one per element (x's shape) or per row (x's shape with a last dimension of 1).  scale:
    D elements, or one; with post_weight and pre_weight (D elements each) in one type, fp32 or bf16.  Returns h in x's type
    and y in block's.  y is formed from h before h is rounded.  Rows may have any distance from each other.  D is at
    most 16384.  Every input has a gradient; sums over rows are fp32 in a fixed order."""
    tensors = [("x", x), ("block", block), ("post_weight", post_weight), ("pre_weight", pre_weight)]
    tensors += [(n, t) for n, t in (("gate", gate), ("scale", scale)) if t is not None]
    for name, t in tensors:
        require_gpu_tensor(t, name)
        _dtype(t, name)
        if t.device != x.device:
            raise _lib.MuonAmdError(f"{name} is on {t.device}, x on {x.device}")
    if x.ndim < 1 or block.shape != x.shape:
        raise ValueError(f"block must have the shape of x, {tuple(x.shape)}, got {tuple(block.shape)}")
    width, limit = x.size(-1), _lib.load().muon_amd_residual_norm_max_width()
    if width > limit:
        raise ValueError(f"rows of {width} channels: at most {limit} are taken")
    if x.dtype == torch.bfloat16 and block.dtype != torch.bfloat16:
        raise TypeError("a bf16 residual stream takes a bf16 block")
    for name, t in (("post_weight", post_weight), ("pre_weight", pre_weight)):
        if t.shape != (width,):
            raise ValueError(f"{name} must have {width} elements, got {tuple(t.shape)}")
    if scale is not None and (scale.ndim > 1 or scale.numel() not in (1, width)):
        raise ValueError(f"scale must have {width} elements or one, got {tuple(scale.shape)}")
    if pre_weight.dtype != post_weight.dtype or (scale is not None and scale.dtype != post_weight.dtype):
        raise TypeError("post_weight, pre_weight and scale must have one type")
    if gate is not None:
        if gate.shape not in (x.shape, x.shape[:-1] + (1,)):
            raise ValueError(f"gate must have the shape {tuple(x.shape)} or {tuple(x.shape[:-1]) + (1,)}, got {tuple(gate.shape)}")
        if gate.dtype != block.dtype:
            raise TypeError(f"gate is {gate.dtype}, block {block.dtype}: they must have one type")
    if not eps >= 0.0:
        raise ValueError(f"eps must not be negative, got {eps}")
    return _ResidualNorm.apply(x, block, post_weight, pre_weight, gate, scale, float(eps))


class Routing(NamedTuple):
    """What route_topk returns."""
    weights: torch.Tensor        # (..., k) fp32
    indices: torch.Tensor        # (..., k) int32, -1 where a choice is not there
    counts: torch.Tensor         # (experts,) int32
    balance_loss: torch.Tensor   # 0-dim fp32
    z_loss: torch.Tensor         # 0-dim fp32


class _RouteTopk(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, k, mask, normalize):
        experts = logits.size(-1)
        tokens = logits.numel() // experts
        f32 = lambda *shape: torch.empty(shape, dtype=torch.float32, device=logits.device)
        weights, indices = f32(*logits.shape[:-1], k), torch.empty(*logits.shape[:-1], k, dtype=torch.int32, device=logits.device)
        ctx.set_materialize_grads(False)
        ctx.normalize = normalize
        if tokens == 0:
            counts, balance, z = torch.zeros(experts, dtype=torch.int32, device=logits.device), f32().zero_(), f32().zero_()
            ctx.save_for_backward(logits, None, None, None, None, None, None)
        else:
            counts, balance, z = torch.empty(experts, dtype=torch.int32, device=logits.device), f32(), f32()
            part, lse = f32(), f32(tokens)
            lib = _lib.load()
            partials = f32(lib.muon_amd_route_partials(tokens, experts))
            a, keep = _route_args(logits, mask, weights, indices, counts, part, lse, normalize)
            a.balance, a.z, a.partials = balance.data_ptr(), z.data_ptr(), partials.data_ptr()
            with torch.cuda.device(logits.device):
                _launch("route", logits.numel() * logits.element_size() + 8 * indices.numel(), lambda: _lib.check(
                    lib.muon_amd_route(ctypes.byref(a), _stream_ptr(logits.device)), "route"))
            if ctx.needs_input_grad[0]:
                ctx.save_for_backward(logits, mask, weights, indices, counts, part, lse)
        ctx.mark_non_differentiable(indices, counts)
        return weights, indices, counts, balance, z

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dweights, _, __, dbalance, dz):
        logits, mask, weights, indices, counts, part, lse = ctx.saved_tensors
        dlogits = torch.empty(logits.shape, dtype=logits.dtype, device=logits.device)
        if lse is None:
            return dlogits, None, None, None
        a, keep = _route_args(logits, mask, weights, indices, counts, part, lse, ctx.normalize)
        a.dlogits = dlogits.data_ptr()
        if dweights is not None:
            dweights = _rows(dweights, a.k)
            a.dweights, a.ld_dweights = dweights.data_ptr(), dweights.stride(0)
        a.dbalance, a.dz = (None if t is None else t.data_ptr() for t in (dbalance, dz))
        with torch.cuda.device(logits.device):
            _launch("route_backward", 2 * logits.numel() * logits.element_size() + 12 * indices.numel(), lambda: _lib.check(
                _lib.load().muon_amd_route_backward(ctypes.byref(a), _stream_ptr(logits.device)), "route_backward"))
        return dlogits, None, None, None


def _route_args(logits, mask, weights, indices, counts, part, lse, normalize):
    """The arguments of both directions, and the tensors behind the addresses in them."""
    rows = _rows(logits, logits.size(-1))
    flags = None if mask is None else mask.contiguous()
    a = _lib.RouteArgs(logits=rows.data_ptr(), mask=None if flags is None else flags.data_ptr(), weights=weights.data_ptr(),
                       indices=indices.data_ptr(), counts=counts.data_ptr(), part=part.data_ptr(), lse=lse.data_ptr(), tokens=rows.size(0),
                       ld_logits=rows.stride(0), experts=rows.size(1), k=weights.size(-1), dtype=_DTYPES[logits.dtype],
                       normalize=int(normalize))
    return a, (rows, flags)


def route_topk(logits: torch.Tensor, k: int, *, mask: torch.Tensor | None = None, normalize: bool = True) -> Routing:
    """The k experts of each token from its logits (..., experts), fp32 or bf16, with the losses of a balanced router:

        p = softmax(logits);  indices: the k largest logits, of equal ones the lowest index first
        weights = p at indices, divided by their sum (normalize=False: as they are)
        counts[e] = tokens that have e among their k
        balance_loss = E sum_e (counts[e] / (N k)) (mean of p[:, e]);  z_loss = mean of logsumexp(logits)^2

    over the N tokens that take part: those whose `mask` (bool, the shape of logits without its last dimension) is true and
    that have an expert available at all.  An expert whose logit is -infinity is not available to that token; a
    choice that is not there has index -1 and weight 0.  A token that takes no part has indices -1, weights 0 and no
    gradient.  Gradients flow to the logits from weights, balance_loss (through p; counts are constants) and z_loss.
    NaN counts as the largest logit.  At most 1024 experts and 32 choices.  Sums are fp32 in a fixed order."""
    require_gpu_tensor(logits, "logits")
    _dtype(logits, "logits")
    lib = _lib.load()
    if logits.ndim < 1 or not 1 <= logits.size(-1) <= lib.muon_amd_route_max_experts():
        raise ValueError(f"logits must have 1 to {lib.muon_amd_route_max_experts()} experts as their last dimension, got {tuple(logits.shape)}")
    if isinstance(k, bool) or int(k) != k or not 1 <= k <= min(logits.size(-1), lib.muon_amd_route_max_k()):
        raise ValueError(f"k must be 1 to {min(logits.size(-1), lib.muon_amd_route_max_k())}, got {k!r}")
    if mask is not None:
        require_gpu_tensor(mask, "mask")
        if mask.dtype != torch.bool or mask.shape != logits.shape[:-1] or mask.device != logits.device:
            raise ValueError(f"mask must be a bool tensor of shape {tuple(logits.shape[:-1])} on {logits.device}, got {mask.dtype} {tuple(mask.shape)}")
    return Routing(*_RouteTopk.apply(logits, int(k), mask, bool(normalize)))
