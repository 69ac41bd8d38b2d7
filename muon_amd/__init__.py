"""muon_amd -- the Muon optimizer step for AMD Instinct MI355X (gfx950).

Drop-in for the single-GPU surface of the reference `muon` module: the same class and function
names, argument order, defaults and optimizer state keys, with the device work done by
hand-written HIP kernels in libmuon_amd.so (see include/muon_amd.h for its C ABI).
"""
from .functional import (adam_update, clear_engine_cache, muon_update, zeropower_via_aol4,
                         zeropower_via_newtonschulz5)
from .gradients import clip_coefficient, clip_grad_norm_
from .layers import Routing, residual_norm, route_topk
from .losses import CrossEntropy, distill_topk, linear_cross_entropy
from .ops import ns_line_1, ns_line_2, ns_line_3
from .optim import AdamW, Muon, MuonWithAuxAdam, SingleDeviceMuon, SingleDeviceMuonWithAuxAdam
from ._lib import MuonAmdError

__all__ = [
    "Muon", "SingleDeviceMuon", "MuonWithAuxAdam", "SingleDeviceMuonWithAuxAdam",
    "zeropower_via_newtonschulz5", "zeropower_via_aol4", "muon_update", "adam_update", "clear_engine_cache",
    "ns_line_1", "ns_line_2", "ns_line_3",
    "AdamW", "clip_grad_norm_", "clip_coefficient", "residual_norm", "route_topk", "Routing",
    "linear_cross_entropy", "CrossEntropy", "distill_topk",
    "MuonAmdError",
]
