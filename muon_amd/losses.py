"""What a language model is trained on, as torch functions with gradients.

    linear_cross_entropy(hidden, weight, targets)  -> loss, lse
        the cross entropy of a linear head over a large vocabulary, without keeping its logits
    distill_topk(logits, teacher_logits, teacher_indices, temperature=...)  -> loss
        distillation from the largest logits of a teacher
"""
from __future__ import annotations

from typing import NamedTuple

import torch

from . import _lib
from .engine import require_gpu_tensor
from .layers import _dtype, _no_tangent


def _reduction(reduction) -> int:
    """The reduction's number, or -1 for what is none."""
    return _lib.REDUCTIONS.get(reduction, -1) if isinstance(reduction, str) else -1


def _refuse_reduction(reduction):
    if _reduction(reduction) < 0:
        raise ValueError(f"reduction must be one of {', '.join(sorted(_lib.REDUCTIONS))}, got {reduction!r}")


class CrossEntropy(NamedTuple):
    """What linear_cross_entropy returns."""
    loss: torch.Tensor           # 0-dim fp32, or (reduction="none") one for each token
    lse: torch.Tensor            # log sum exp of each token's logits, fp32


def linear_cross_entropy(hidden: torch.Tensor, weight: torch.Tensor, targets: torch.Tensor, *, ignore_index: int = -100,
                         reduction: str = "mean") -> CrossEntropy:
    """The loss of a linear head without its logits in memory: hidden (..., D) bf16, weight (V, D) bf16, targets (...) int32 or
    int64, and with x = hidden weight^T

        lse = log sum exp(x) over the V classes;  loss = lse - x[target]

    as the mean over the tokens that take part (zero where none does), their "sum", or ("none") of each token, fp32.  lse is
    there for every token and has a gradient of its own: lse.square() in the objective is the z-loss of a head.  A token whose target is
    ignore_index takes no part: its loss, lse and gradient are zero and its hidden state may hold anything; the products leave it
    out.  Any other target outside of 0 .. V - 1 gives a loss that is not a number, and such gradients.

    The products are of bf16 numbers with fp32 sums.  Backward forms the logits again in pieces of the vocabulary, rounds their gradient to
    bf16 once, and returns both gradients in bf16.  There are at most 2^24 tokens and classes, 65536 channels, and fewer than 2^39 logits (in whole
    tiles of 256 x 256).  Infinities in the matrix may leave gradients that are no numbers (zero times infinity).  The same call gives the same bits.
    Workspaces: forward 8 bytes for 256 logits (128 where there are few), backward at most 1 GiB for the logits' gradient (4096 of its columns
    where there are more than 131072 tokens) and half a GiB or 4 D bytes a token, whichever is more, for sums; both 2 D bytes a token, a
    copy of the matrix unless D is a multiple of 64 and its rows lie at multiples of 16 bytes, and one before that unless its channels lie next to each other."""
    if isinstance(ignore_index, int) and not isinstance(ignore_index, bool) and -1 << 63 <= ignore_index < 1 << 63:
        out = _lib.native().linear_cross_entropy(hidden, weight, targets, ignore_index, _reduction(reduction))
        if out is not None:
            return CrossEntropy(*out)
    _refuse_head(hidden, weight, targets, ignore_index, reduction)


def _refuse_head(hidden, weight, targets, ignore_index, reduction):
    """Says what is wrong with arguments that were not taken."""
    for name, t in (("hidden", hidden), ("weight", weight)):
        require_gpu_tensor(t, name)
        if t.dtype != torch.bfloat16:
            raise TypeError(f"{name} is {t.dtype}: bf16 tensors are taken")
    require_gpu_tensor(targets, "targets")
    if targets.dtype not in (torch.int32, torch.int64):
        raise TypeError(f"targets is {targets.dtype}: int32 and int64 are taken")
    for name, t in (("weight", weight), ("targets", targets)):
        if t.device != hidden.device:
            raise _lib.MuonAmdError(f"{name} is on {t.device}, hidden on {hidden.device}")
    if hidden.ndim < 1 or not 1 <= hidden.size(-1) <= 1 << 16:
        raise ValueError(f"hidden must have 1 to 65536 channels as its last dimension, got {tuple(hidden.shape)}")
    if weight.ndim != 2 or weight.size(1) != hidden.size(-1) or not 1 <= weight.size(0) <= 1 << 24:
        raise ValueError(f"weight must have 1 to 2^24 rows of {hidden.size(-1)} channels, got {tuple(weight.shape)}")
    if targets.shape != hidden.shape[:-1] or targets.numel() > 1 << 24:
        raise ValueError(f"targets must have the shape {tuple(hidden.shape[:-1])} and at most 2^24 elements, got {tuple(targets.shape)}")
    if not isinstance(ignore_index, int) or isinstance(ignore_index, bool) or not -1 << 63 <= ignore_index < 1 << 63:
        raise ValueError(f"ignore_index must be a whole number of 64 bits, got {ignore_index!r}")
    _refuse_reduction(reduction)
    _no_tangent(hidden, "hidden")
    _no_tangent(weight, "weight")
    raise _lib.MuonAmdError("linear_cross_entropy does not take these arguments")


def distill_topk(logits: torch.Tensor, teacher_logits: torch.Tensor, teacher_indices: torch.Tensor, *, temperature: float = 1.0,
                 mask: torch.Tensor | None = None, reduction: str = "mean") -> torch.Tensor:
    """Distillation of a student, logits (..., vocabulary) in fp32 or bf16, from the largest logits that a teacher kept for
    each token: teacher_logits (..., k), fp32 or bf16, at teacher_indices (..., k), int32 or int64, T = temperature:

        p = softmax(logits / T) over the vocabulary;  q = softmax(teacher_logits / T) over the token's list
        loss = T^2 sum_k q_k (log q_k - log p[teacher_indices_k])

    as the mean over the tokens that take part (zero where none does), their "sum", or ("none") of each token, fp32; T from 1e-15 to 1e15.  Entries
    whose index is outside of the vocabulary (-1 by habit) or whose teacher logit is -infinity are not there; a token whose
    list has none, or whose `mask` (bool, the shape of logits without its last dimension) is false, takes no part: its loss and
    gradient are zero, whatever its logits hold.  An index that comes several times counts with the sum of its
    q.  The gradient flows to logits alone.  At most 1024 entries a token, fewer than 2^24 tokens; where
    a gradient is wanted, fewer than 2^24 pieces of 16 KiB that the tokens' logits take (a row takes whole ones).  Sums are fp32 in a fixed order."""
    if isinstance(temperature, (int, float)):
        out = _lib.native().distill_topk(logits, teacher_logits, teacher_indices, float(temperature), mask, _reduction(reduction))
        if out is not None:
            return out
    _refuse_distill(logits, teacher_logits, teacher_indices, temperature, mask, reduction)


def _refuse_distill(logits, teacher_logits, teacher_indices, temperature, mask, reduction):
    """Says what is wrong with arguments that were not taken."""
    for name, t in (("logits", logits), ("teacher_logits", teacher_logits)):
        require_gpu_tensor(t, name)
        _dtype(t, name)
    require_gpu_tensor(teacher_indices, "teacher_indices")
    if teacher_indices.dtype not in (torch.int32, torch.int64):
        raise TypeError(f"teacher_indices is {teacher_indices.dtype}: int32 and int64 are taken")
    for name, t in (("teacher_logits", teacher_logits), ("teacher_indices", teacher_indices)):
        if t.device != logits.device:
            raise _lib.MuonAmdError(f"{name} is on {t.device}, logits on {logits.device}")
    if logits.ndim < 1 or not 1 <= logits.size(-1) <= 1 << 30:
        raise ValueError(f"logits must have 1 to 2^30 classes as their last dimension, got {tuple(logits.shape)}")
    limit = _lib.load().muon_amd_distill_max_top()
    if teacher_logits.ndim != logits.ndim or teacher_logits.shape[:-1] != logits.shape[:-1] or not 1 <= teacher_logits.size(-1) <= limit:
        raise ValueError(f"teacher_logits must be {tuple(logits.shape[:-1])} lists of 1 to {limit} entries, got {tuple(teacher_logits.shape)}")
    if teacher_indices.shape != teacher_logits.shape:
        raise ValueError(f"teacher_indices must have the shape of teacher_logits, {tuple(teacher_logits.shape)}, got {tuple(teacher_indices.shape)}")
    if logits.numel() // logits.size(-1) >= 1 << 24:
        raise ValueError(f"{logits.numel() // logits.size(-1)} tokens: fewer than 2^24 are taken")
    if mask is not None:
        require_gpu_tensor(mask, "mask")
        if mask.dtype != torch.bool or mask.shape != logits.shape[:-1] or mask.device != logits.device:
            raise ValueError(f"mask must be a bool tensor of shape {tuple(logits.shape[:-1])} on {logits.device}, got {mask.dtype} {tuple(mask.shape)}")
    if not isinstance(temperature, (int, float)) or not 1e-15 <= temperature <= 1e15:
        raise ValueError(f"temperature must be a number from 1e-15 to 1e15, got {temperature!r}")
    _refuse_reduction(reduction)
    _no_tangent(logits, "logits")
    _no_tangent(teacher_logits, "teacher_logits")
    if torch.is_grad_enabled() and teacher_logits.requires_grad:
        raise ValueError("teacher_logits requires a gradient: there is none for the teacher (detach it)")
    raise _lib.MuonAmdError("distill_topk does not take these arguments")
