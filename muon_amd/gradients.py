"""The norm of all gradients of a model and clipping by it, as grouped launches over the gradients.

    clip_grad_norm_(parameters, max_norm)       scales the gradients in place, as torch.nn.utils' function of that name
    clip_coefficient(parameters, max_norm)      -> (norm, coefficient); the coefficient goes to AdamW.step(grad_scale=...),
                                                which then scales on the way: one pass over the gradients less

norm = sqrt(sum of squares over every element), coefficient = min(1, max_norm / (norm + 1e-6)).  Squares and sums are
formed in 64 bits and rounded once to fp32, in a fixed order.  Nothing waits for the device (except error_if_nonfinite).
"""
from __future__ import annotations

from collections import OrderedDict

import numpy as np
import torch

from . import _lib, plan as _plan
from .engine import _launch, _Staging, _stream_ptr, _upload, require_gpu_tensor
from .functional import _cached, _exclusive, _src_dtype

_GRAD_CACHE_MAX = 16      # tables of gradient lists: small
_GRAD_CACHE: "OrderedDict[tuple, object]" = OrderedDict()


class _GradList:
    """Descriptor table, block prefix and workspace for the gradients of a list of sizes and types."""

    def __init__(self, numels, dtypes, device):
        self.device = device
        self.descs = np.zeros(len(numels), dtype=_lib.GRAD_DESC)
        self.descs["numel"], self.descs["dtype"] = numels, dtypes
        self.prefix = _plan.adam_block_prefix(numels)
        self.nblocks = int(self.prefix[-1])
        self.nbytes = int(sum(n * (2 if t == _lib.SRC_BF16 else 4) for n, t in zip(numels, dtypes)))
        self.prefix_dev = _upload(self.prefix, device)
        self.desc_dev = torch.empty(self.descs.nbytes, dtype=torch.uint8, device=device)
        self.partials = torch.empty(_lib.load().muon_amd_grad_norm_partials(), dtype=torch.float64, device=device)
        self.staging = _Staging(device)
        self.key = None

    def run(self, pointers, max_norm, in_place):
        """pointers: the gradients' addresses as the bytes of 64-bit numbers."""
        lib = _lib.load()
        if pointers != self.key:
            self.descs["grad"] = np.frombuffer(pointers, dtype=np.uint64)
            _lib.check(lib.muon_amd_validate_grads(_lib.host_ptr(self.descs), len(self.descs), _lib.host_ptr(self.prefix)), "validate_grads")
            self.staging.upload(self.descs, self.desc_dev)
            self.key = pointers
        out = torch.empty(2, dtype=torch.float32, device=self.device)
        call = lib.muon_amd_grad_clip if in_place else lib.muon_amd_grad_norm
        _launch("grad_clip" if in_place else "grad_norm", self.nbytes * (3 if in_place else 1), lambda: _lib.check(call(
            self.desc_dev.data_ptr(), self.prefix_dev.data_ptr(), len(self.descs), self.nblocks, self.partials.data_ptr(),
            max_norm, out.data_ptr(), _stream_ptr(self.device)), "grad_norm"))
        return out[0], out[1]


def _general_rows(parameters, writebacks):
    """What _native.gradient_rows gives for plain gradients: (device index, sizes and types, addresses, the tensors behind
    them); other strides go through contiguous copies."""
    grads, seen = [], set()
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
            c = g.contiguous()
            writebacks.append((g, c))
            g = c
        if g.numel():
            grads.append(g)
    if not grads:
        return None
    if any(g.device != grads[0].device for g in grads):
        raise _lib.MuonAmdError("the gradients must be on one device")
    kinds = np.array([(g.numel(), _src_dtype(g)) for g in grads], dtype=np.int64)
    return grads[0].device.index, kinds.tobytes(), np.array([g.data_ptr() for g in grads], dtype=np.uint64).tobytes(), grads


def _clip(parameters, max_norm, in_place):
    parameters = [parameters] if isinstance(parameters, torch.Tensor) else list(parameters)
    max_norm = float(max_norm)
    if not max_norm >= 0.0:
        raise ValueError(f"max_norm must not be negative, got {max_norm}")
    writebacks = []
    rows = _lib.native().gradient_rows(parameters) or _general_rows(parameters, writebacks)
    if rows is None:
        device = parameters[0].device if parameters else "cpu"
        return torch.zeros((), device=device), torch.ones((), device=device)
    index, kinds, pointers = rows[:3]
    device = torch.device("cuda", index)

    def make():
        sizes = np.frombuffer(kinds, dtype=np.int64).reshape(-1, 2)
        return _GradList(sizes[:, 0], sizes[:, 1], device)

    with torch.cuda.device(device):
        table = _cached(("grads", index, kinds), make, _GRAD_CACHE, _GRAD_CACHE_MAX)
        with _exclusive(table, device):
            result = table.run(pointers, max_norm, in_place)
    if in_place:
        for dst, src in writebacks:
            dst.copy_(src)
    return result


@torch.no_grad()
def clip_coefficient(parameters, max_norm: float):
    """(norm, coefficient) of the gradients of `parameters` (a tensor or an iterable; those without a gradient are left
    out) as 0-dim fp32 tensors on their device.  A norm that is not finite gives the coefficient that this formula gives
    (zero, or not a number)."""
    return _clip(parameters, max_norm, False)


@torch.no_grad()
def clip_grad_norm_(parameters, max_norm: float, error_if_nonfinite: bool = False) -> torch.Tensor:
    """Scales the gradients in place so that their joint 2-norm is at most max_norm; returns the norm before that as a
    0-dim fp32 tensor.  Gradients whose norm is small enough are not written.  error_if_nonfinite raises before anything
    is scaled if the norm is infinite or not a number, and waits for the device to know."""
    if error_if_nonfinite:
        parameters = [parameters] if isinstance(parameters, torch.Tensor) else list(parameters)
        norm, _ = _clip(parameters, max_norm, False)
        if not bool(torch.isfinite(norm)):
            raise RuntimeError(f"the total norm of the gradients is {float(norm)}, so they cannot be clipped")
    return _clip(parameters, max_norm, True)[0]
