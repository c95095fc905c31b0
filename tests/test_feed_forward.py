"""Refusals of the feed-forward operators, on the CPU: every wrong argument ends in an error before
any CUDA call."""
import ctypes

import pytest
import torch

ONE = ctypes.c_void_p(256)


def test_rms_norm_c_refusals():
    from ae_mlsys_gnn_b200 import _capi

    lib = _capi.lib()
    fwd = lambda **k: lib.gnn_rms_norm_fwd(k.get("x", ONE), None, ONE, k.get("dtype", 1), k.get("wdtype", 1),
                                           k.get("n", 4), k.get("d", 8), 1e-6, k.get("y", ONE), None, None, None)
    assert fwd(n=0) == 0
    assert fwd(x=None) == -1 and "null" in _capi.last_error()
    assert fwd(y=None) == -1 and fwd(n=-1) == -1 and fwd(d=0) == -1
    assert fwd(dtype=3) == -4 and fwd(dtype=1, wdtype=2) == -4 and fwd(dtype=0, wdtype=1) == -4
    assert fwd(d=32769) == -5 and "32768" in _capi.last_error()
    assert lib.gnn_rms_norm_fp8(ONE, None, ONE, 1, 1, 4, 8, 1e-6, 64, ONE, ONE, None, None) == -4
    assert lib.gnn_rms_norm_fp8(ONE, None, ONE, 1, 1, 4, 8, 1e-6, 0, None, ONE, None, None) == -1
    assert lib.gnn_rms_norm_fp8(ONE, None, ONE, 1, 1, 4, 8, 1e-6, 0, ONE, None, None, None) == -1
    need = ctypes.c_size_t(0)
    assert lib.gnn_rms_norm_bwd_workspace_bytes(100, 64, ctypes.byref(need)) == 0 and need.value >= 100 * 64 * 4
    assert lib.gnn_rms_norm_bwd_workspace_bytes(-1, 64, ctypes.byref(need)) == -1
    bwd = lambda ws, nb: lib.gnn_rms_norm_bwd(ONE, None, ONE, ONE, ONE, 1, 1, 100, 64, ONE, ONE, ws, nb, None)
    assert bwd(None, 1 << 20) == -3 and bwd(ONE, need.value - 1) == -3
    assert lib.gnn_rms_norm_bwd(None, None, ONE, ONE, ONE, 1, 1, 100, 64, ONE, ONE, ONE, 1 << 20, None) == -1


def test_rms_norm_refuses_cpu_tensors():
    from ae_mlsys_gnn_b200.operators.rms_norm import add_rms_norm, add_rms_norm_fp8

    for f in (add_rms_norm, add_rms_norm_fp8):
        with pytest.raises(ValueError, match="CUDA"):
            f(torch.zeros(2, 4), torch.ones(4))
        with pytest.raises(TypeError):
            f([1.0], torch.ones(4))
