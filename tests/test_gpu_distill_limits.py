"""The largest launches of distill_topk: what its backward pass would refuse is refused before a loss is returned."""
import ctypes

import pytest
import torch

import muon_amd
from muon_amd import _lib

DEV = "cuda:0"
ROWS = 1 << 23                 # of two pieces each: one launch forward, one too many backward


@pytest.mark.parametrize("dtype,vocab", [(_lib.SRC_F32, 4097), (_lib.SRC_BF16, 8193)])
def test_a_gradient_that_no_launch_holds_is_refused_forward(dtype, vocab):
    lib = _lib.load()
    pointers = ("logits", "teacher", "indices", "losses", "part", "stats", "partials", "counter", "dloss", "dlogits")
    good = dict({p: 4096 for p in pointers}, tokens=ROWS, ld_logits=vocab, ld_teacher=2, ld_indices=2, vocab=vocab, top=2, dtype=dtype, teacher_dtype=dtype,
                index_bits=32, temperature=1.0)
    assert lib.muon_amd_distill(ctypes.byref(_lib.DistillArgs(**good, differentiable=1)), None) == -1
    assert "more than a launch holds" in lib.muon_amd_last_error().decode()
    assert lib.muon_amd_distill_backward(ctypes.byref(_lib.DistillArgs(**good)), None) == -1


@pytest.mark.gpu
def test_many_rows_of_two_pieces():
    logits = torch.zeros(1, 4097, device=DEV).expand(ROWS, 4097)
    teacher, at = torch.zeros(1, 1, device=DEV).expand(ROWS, 1), torch.zeros(1, 1, dtype=torch.int32, device=DEV).expand(ROWS, 1)
    loss = muon_amd.distill_topk(logits, teacher, at)                # without a gradient it is one launch
    assert abs(float(loss) - 8.318) < 1e-2                           # (log 4097; a sum of 2^23 of them)
    with pytest.raises(muon_amd.MuonAmdError, match="more than a launch holds"):
        muon_amd.distill_topk(logits.detach().requires_grad_(), teacher, at)
    # one piece fewer than 2^24
    leaf = logits[:, :4096].detach().requires_grad_()
    assert abs(float(muon_amd.distill_topk(leaf, teacher, at).detach()) - 8.318) < 1e-2


@pytest.mark.gpu
def test_too_many_tokens():
    rows = 1 << 24
    one = torch.zeros(1, 8, device=DEV)
    with pytest.raises(ValueError, match="fewer than 2"):
        muon_amd.distill_topk(one.expand(rows, 8), one[:, :1].expand(rows, 1), torch.zeros(1, 1, dtype=torch.int32, device=DEV).expand(rows, 1))
    loss = muon_amd.distill_topk(one.expand(rows - 1, 8), one[:, :1].expand(rows - 1, 1), torch.zeros(1, 1, dtype=torch.int32, device=DEV).expand(rows - 1, 1), reduction="none")
    assert loss.shape == (rows - 1,) and float((loss - 2.0794415).abs().max()) <= 1e-5
