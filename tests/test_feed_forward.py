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


def test_experts_c_refusals():
    from ae_mlsys_gnn_b200 import _capi

    lib = _capi.lib()
    need = ctypes.c_size_t(1)
    size = lambda n, e: lib.gnn_expert_sort_workspace_bytes(n, e, ctypes.byref(need))
    assert size(2048, 64) == 0 and need.value == 0  # one chunk: no scratch
    assert size(1 << 20, 64) == 0 and 0 < need.value <= 148 * 64 * 4 + 16
    assert size(-1, 64) == -1 and size(5, 0) == -1
    sort = lambda n=1 << 20, e=64, ids=ONE, ws=ONE, nb=1 << 30: lib.gnn_expert_sort(ids, 0, n, e, ONE, ONE, ws, nb, None)
    assert sort(ws=None) == -3 and sort(nb=100) == -3
    assert sort(e=1025) == -5 and sort(n=1 << 31) == -5
    assert sort(ids=None) == -1 and sort(n=-1) == -1
    disp = lambda x=ONE, dt=1, t=4, k=2, d=8: lib.gnn_expert_dispatch(x, ONE, ONE, dt, t, k, d, ONE, None)
    assert disp(t=0) == 0
    assert disp(x=None) == -1 and disp(k=0) == -1 and disp(d=0) == -1 and disp(t=-1) == -1
    assert disp(dt=7) == -4 and disp(k=33) == -5 and disp(t=1 << 30, k=4) == -5
    comb = lambda rows=ONE, dt=1, wdt=1: lib.gnn_expert_combine(rows, None, ONE, dt, wdt, 4, 2, 8, ONE, None)
    assert comb(rows=None) == -1 and comb(dt=1, wdt=2) == -4 and comb(dt=0, wdt=1) == -4
    assert lib.gnn_expert_combine_bwd(ONE, ONE, None, ONE, ONE, 1, 1, 4, 2, 8, ONE, ONE, None) == -1


def test_experts_refuse_cpu_tensors():
    from ae_mlsys_gnn_b200.operators.experts import expert_sort

    with pytest.raises(ValueError, match="CUDA"):
        expert_sort(torch.zeros(4, 2, dtype=torch.int32), 3)
    with pytest.raises(TypeError):
        expert_sort([[0]], 3)
