"""The norm of all gradients of a model and clipping by it, as grouped launches over the gradients.

    clip_grad_norm_(parameters, max_norm)       scales the gradients in place, as torch.nn.utils' function of that name
    clip_coefficient(parameters, max_norm)      -> (norm, coefficient); the coefficient goes to AdamW.step(grad_scale=...),
                                                which then scales on the way: one pass over the gradients less

norm = sqrt(sum of squares over every element), coefficient = min(1, max_norm / (norm + 1e-6)).  Squares and sums are
formed in 64 bits and rounded once to fp32, in a fixed order.  Nothing waits for the device (except error_if_nonfinite).
"""
from __future__ import annotations

import torch

from . import _lib, engine as _engine
from .engine import _launch, require_gpu_tensor


def _general(parameters, max_norm, in_place):
    """Gradients that are not all row-major, or a list that is to be refused."""
    grads, writebacks, seen = [], [], set()
    for p in parameters:
        g = p.grad
        if g is None:
            continue
        require_gpu_tensor(g, "gradient")
        if g.is_sparse or g.dtype not in (torch.float32, torch.bfloat16):
            raise NotImplementedError(f"muon_amd clips dense fp32 and bf16 gradients; got {g.dtype}{' (sparse)' if g.is_sparse else ''}")
        if id(p) in seen:
            raise ValueError("the same parameter is in the list twice")
        seen.add(id(p))
        if not g.is_contiguous():                 # the kernels address row-major memory
            if in_place and any(n > 1 and st == 0 for n, st in zip(g.shape, g.stride())):
                raise ValueError("gradients that share memory cannot be scaled in place (one is broadcast)")
            c = g.contiguous()
            writebacks.append((g, c))
            g = c
        if g.numel():
            grads.append(g)
    if not grads:
        device = parameters[0].device if parameters else "cpu"
        return torch.zeros((), device=device), torch.ones((), device=device)
    if any(g.device != grads[0].device for g in grads):
        raise _lib.MuonAmdError("the gradients must be on one device")
    result = _lib.native().clip_list(grads, max_norm, in_place)
    if in_place:
        for dst, src in writebacks:
            dst.copy_(src)
    return result


def _clip(parameters, max_norm, in_place):
    parameters = [parameters] if isinstance(parameters, torch.Tensor) else list(parameters)
    max_norm = float(max_norm)
    if not max_norm >= 0.0:
        raise ValueError(f"max_norm must not be negative, got {max_norm}")
    native = _lib.native()
    if _engine.PROFILE is None:
        result = native.clip(parameters, max_norm, in_place)
        return result if result is not None else _general(parameters, max_norm, in_place)
    out = []
    nbytes = sum(p.grad.numel() * p.grad.element_size() for p in parameters if p.grad is not None)
    _launch("grad_clip" if in_place else "grad_norm", nbytes * (3 if in_place else 1),
            lambda: out.append(native.clip(parameters, max_norm, in_place) or _general(parameters, max_norm, in_place)))
    return out[0]


def clip_coefficient(parameters, max_norm: float):
    """(norm, coefficient) of the gradients of `parameters` (a tensor or an iterable; those without a gradient are left
    out) as 0-dim fp32 tensors on their device.  A norm that is not finite gives the coefficient that this formula gives
    (zero, or not a number)."""
    with torch.no_grad():
        return _clip(parameters, max_norm, False)


def clip_grad_norm_(parameters, max_norm: float, error_if_nonfinite: bool = False) -> torch.Tensor:
    """Scales the gradients in place so that their joint 2-norm is at most max_norm; returns the norm before that as a
    0-dim fp32 tensor.  Gradients whose norm is small enough are not written; ones that share memory are refused.  error_if_nonfinite raises before anything
    is scaled if the norm is infinite or not a number, and waits for the device to know."""
    with torch.no_grad():
        if error_if_nonfinite:
            parameters = [parameters] if isinstance(parameters, torch.Tensor) else list(parameters)
            norm, _ = _clip(parameters, max_norm, False)
            if not bool(torch.isfinite(norm)):
                raise RuntimeError(f"the total norm of the gradients is {float(norm)}, so they cannot be clipped")
        return _clip(parameters, max_norm, True)[0]
