"""Operators of a transformer's forward and backward pass whose weights the optimizers of this package train, as torch
functions with gradients.

    residual_norm(x, block, post_weight, pre_weight, gate=..., scale=...)  -> h, y
        the norm after a block, its gate and residual scale, the addition to the residual stream, and the norm before
        the next block, in one pass
    route_topk(logits, k)  -> weights, indices, counts, balance_loss, z_loss
        the experts of each token, tokens per expert, and the losses that keep them balanced
"""
from __future__ import annotations

from typing import NamedTuple

import torch

from . import _lib
from .engine import require_gpu_tensor

_DTYPES = {torch.float32: _lib.SRC_F32, torch.bfloat16: _lib.SRC_BF16}


def _dtype(t: torch.Tensor, name: str) -> int:
    try:
        return _DTYPES[t.dtype]
    except KeyError:
        raise TypeError(f"{name} is {t.dtype}: fp32 and bf16 tensors are taken") from None


def _no_tangent(t: torch.Tensor, name: str) -> None:
    if torch.autograd.forward_ad.unpack_dual(t).tangent is not None:
        raise NotImplementedError(f"{name} carries a forward-mode derivative: only gradients (reverse mode) are there")


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
    out = _lib.native().residual_norm(x, block, post_weight, pre_weight, gate, scale, eps)
    return out if out is not None else _refuse_residual(x, block, post_weight, pre_weight, gate, scale, eps)


def _refuse_residual(x, block, post_weight, pre_weight, gate, scale, eps):
    """Says what is wrong with arguments that were not taken."""
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
    for name, t in tensors:
        _no_tangent(t, name)
    raise _lib.MuonAmdError("residual_norm does not take these arguments")


class Routing(NamedTuple):
    """What route_topk returns."""
    weights: torch.Tensor        # (..., k) fp32
    indices: torch.Tensor        # (..., k) int32, -1 where a choice is not there
    counts: torch.Tensor         # (experts,) int32
    balance_loss: torch.Tensor   # 0-dim fp32
    z_loss: torch.Tensor         # 0-dim fp32


def route_topk(logits: torch.Tensor, k: int, *, mask: torch.Tensor | None = None, normalize: bool = True, scores: str = "softmax",
               bias: torch.Tensor | None = None, groups: int = 1, groups_kept: int | None = None) -> Routing:
    """The k experts of each token from its logits (..., experts), fp32 or bf16, with the losses of a balanced router:

        p = softmax(logits);  indices: the k largest logits, of equal ones the lowest index first
        weights = p at indices, divided by their sum (normalize=False: as they are)
        counts[e] = tokens that have e among their k
        balance_loss = E sum_e (counts[e] / (N k)) (mean of p[:, e]);  z_loss = mean of logsumexp(logits)^2

    over the N tokens that take part: those whose `mask` (bool, the shape of logits without its last dimension) is true and
    that have an expert available at all.  An expert whose logit is -infinity is not available to that token; a
    choice that is not there has index -1 and weight 0.  A token that takes no part has indices -1, weights 0 and no
    gradient.  Gradients flow to the logits from weights, balance_loss (through p; counts are constants) and z_loss.
    NaN counts as the largest logit.  At most 1024 experts and 32 choices.  Sums are fp32 in a fixed order.

    A router that is balanced without a loss chooses by other numbers than it weighs with:

        s = softmax(logits), or (scores="sigmoid") sigmoid(logits);  c = s + bias
        the experts lie in `groups` equal runs, whose scores are the sums of their two largest c; the `groups_kept` best ones take part
        indices: the k largest c among those, of equal ones the lowest index first;  weights: s at indices, as above

    bias: one fp32 number for each expert, without a gradient (a program raises it for experts with few tokens and lowers it for
    those with many); an expert whose bias is -infinity is not available.  balance_loss is then over s divided by its sum over the
    experts.  What is chosen goes by the order of the c as in 64 bits, not by the rounding of an exponential.  At most 64 groups."""
    if all(isinstance(n, int) and not isinstance(n, bool) for n in (k, groups, 1 if groups_kept is None else groups_kept)):
        kept = groups if groups_kept is None else groups_kept
        out = _lib.native().route_topk(logits, k, mask, bool(normalize), _lib.SCORES.get(scores, -1) if isinstance(scores, str) else -1, bias, groups, kept)
        if out is not None:
            return Routing(*out)
    _refuse_route(logits, k, mask, scores, bias, groups, groups_kept)


def _refuse_route(logits, k, mask, scores, bias, groups, groups_kept):
    """Says what is wrong with arguments that were not taken."""
    require_gpu_tensor(logits, "logits")
    _dtype(logits, "logits")
    lib = _lib.load()
    if logits.ndim < 1 or not 1 <= logits.size(-1) <= lib.muon_amd_route_max_experts():
        raise ValueError(f"logits must have 1 to {lib.muon_amd_route_max_experts()} experts as their last dimension, got {tuple(logits.shape)}")
    if not isinstance(k, int) or isinstance(k, bool) or not 1 <= k <= min(logits.size(-1), lib.muon_amd_route_max_k()):
        raise ValueError(f"k must be 1 to {min(logits.size(-1), lib.muon_amd_route_max_k())}, got {k!r}")
    if mask is not None:
        require_gpu_tensor(mask, "mask")
        if mask.dtype != torch.bool or mask.shape != logits.shape[:-1] or mask.device != logits.device:
            raise ValueError(f"mask must be a bool tensor of shape {tuple(logits.shape[:-1])} on {logits.device}, got {mask.dtype} {tuple(mask.shape)}")
    if not isinstance(scores, str) or scores not in _lib.SCORES:
        raise ValueError(f"scores must be one of {', '.join(sorted(_lib.SCORES))}, got {scores!r}")
    experts, limit = logits.size(-1), lib.muon_amd_route_max_groups()
    if not isinstance(groups, int) or isinstance(groups, bool) or not 1 <= groups <= limit or experts % groups:
        raise ValueError(f"groups must be 1 to {limit} and divide the {experts} experts, got {groups!r}")
    kept = groups if groups_kept is None else groups_kept
    if not isinstance(kept, int) or isinstance(kept, bool) or not 1 <= kept <= groups or k > kept * (experts // groups):
        raise ValueError(f"groups_kept must be 1 to {groups} and leave {k} experts to choose from, got {groups_kept!r}")
    if bias is not None:
        require_gpu_tensor(bias, "bias")
        if bias.dtype != torch.float32:
            raise TypeError(f"bias is {bias.dtype}: fp32 is taken")
        if bias.shape != (experts,) or bias.device != logits.device:
            raise ValueError(f"bias must have {experts} elements on {logits.device}, got {tuple(bias.shape)} on {bias.device}")
        if torch.is_grad_enabled() and bias.requires_grad:
            raise ValueError("bias requires a gradient: there is none (it steers the choice alone)")
        _no_tangent(bias, "bias")
    _no_tangent(logits, "logits")
    raise _lib.MuonAmdError("route_topk does not take these arguments")
