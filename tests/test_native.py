"""The host module of the operators (muon_amd._native): what it says about arguments that it does not take, without a GPU."""
import numpy as np
import pytest
import torch

import muon_amd
from muon_amd import _lib


def test_it_loads_and_is_bound_to_the_library():
    native = _lib.native()
    assert native is _lib.native() and native.abi_version() == _lib.ABI_VERSION


def test_tensors_on_the_host_are_not_taken():
    native = _lib.native()
    z = torch.zeros(4, 8)
    assert native.residual_norm(z, z, z[0], z[0], None, None, 1e-6) is None
    assert native.route_topk(z, 2, None, True) is None
    p = torch.nn.Parameter(torch.zeros(8))
    p.grad = torch.zeros(8)
    assert native.clip([p], 1.0, True) is None and native.clip([], 1.0, True) is None and native.clip([3], 1.0, True) is None
    table = native.AdamWTable([8], [_lib.SRC_F32], 32)
    state = {p: dict(exp_avg=torch.zeros(8), exp_avg_sq=torch.zeros(8), step=0)}
    assert table.collect([p], state) == -1 and table.collect([], state) == -1 and table.collect([p, p], {}) == -1
    assert table.version == 0 and state[p]["step"] == 0
    assert not native.ValueTable().run_plain([p], state, [])


def test_a_missing_module_is_named(monkeypatch):
    import sys
    monkeypatch.setattr(_lib, "_native", None)
    monkeypatch.setitem(sys.modules, "muon_amd._native", None)
    monkeypatch.delattr(muon_amd, "_native", raising=False)
    with pytest.raises(muon_amd.MuonAmdError, match="python -m muon_amd.build"):
        _lib.native()


def test_struct_layouts():
    import ctypes
    lib = _lib.load()
    assert lib.muon_amd_sizeof_adamw_desc() == _lib.ADAMW_DESC.itemsize
    assert lib.muon_amd_sizeof_grad_desc() == _lib.GRAD_DESC.itemsize
    assert lib.muon_amd_sizeof_adamw_values_desc() == 7 * np.dtype("u8").itemsize
    assert lib.muon_amd_sizeof_residual_norm() == ctypes.sizeof(_lib.ResidualNormArgs)
    assert lib.muon_amd_sizeof_route() == ctypes.sizeof(_lib.RouteArgs)
