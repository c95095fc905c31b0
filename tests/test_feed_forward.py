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
    assert size(1024, 64) == 0 and need.value == 0  # one chunk: no scratch
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


def test_linear_c_refusals():
    from ae_mlsys_gnn_b200 import _capi

    lib = _capi.lib()
    BF16, F32, E4M3 = 1, 0, 3

    def fwd(x=ONE, ldx=64, ldw=64, it=BF16, xs=None, ws=None, act=0, y=ONE, ot=BF16, M=4, N=8, K=64, scratch=None, nb=0,
            status=ONE):
        return lib.gnn_linear_fwd(x, ldx, ONE, ldw, it, xs, ws, None, act, 0.2, None, y, None, ot, M, N, K, scratch, nb,
                                  status, None)

    assert fwd(M=0) == 0
    assert fwd(x=None) == -1 and fwd(y=None) == -1 and fwd(status=None) == -1
    assert fwd(M=-1) == -1 and fwd(N=0) == -1 and fwd(K=0) == -1 and fwd(M=1 << 31) == -5
    assert fwd(act=6) == -1 and fwd(act=-1) == -1
    assert fwd(it=4) == -4 and fwd(it=BF16, ot=2) == -4 and fwd(it=E4M3, xs=ONE, ws=ONE, ot=3) == -4
    assert fwd(xs=ONE) == -1 and fwd(it=E4M3) == -1  # scales go with e4m3 operands
    assert fwd(ldx=60) == -1 and fwd(ldw=63) == -1   # a row shorter than K
    assert fwd(M=100, ldx=68) == -4 and fwd(M=100, x=ctypes.c_void_p(264)) == -4  # rows off 16-byte boundaries
    assert fwd(it=F32, ot=F32, ldx=68, M=100) == -4
    assert fwd(it=F32, ot=F32, K=62, ldx=62, ldw=62, M=100) == -4
    assert fwd(it=F32, ot=F32, M=100) == -3  # no scratch
    need = ctypes.c_size_t(0)
    # few rows need no scratch, many rows of a long reduction do
    assert lib.gnn_linear_fwd_workspace_bytes(64, 70, 9000, BF16, ctypes.byref(need)) == 0 and need.value == 0
    assert lib.gnn_linear_fwd_workspace_bytes(300, 70, 9000, BF16, ctypes.byref(need)) == 0 and need.value > 0
    assert fwd(M=300, N=70, K=9000, ldx=9000, ldw=9000) == -3
    assert lib.gnn_linear_fwd_workspace_bytes(64, 70, 9000, 5, ctypes.byref(need)) == -1
    act = lambda gy=ONE, z=ONE, a=4, ldz=8, ws=ONE, nb=1 << 20, gz=ONE, gb=ONE, dt=BF16: lib.gnn_linear_act_bwd(
        gy, z, a, 0.2, dt, 4, 8, gz, ldz, gb, ws, nb, None)
    assert act(gy=None) == -1 and act(z=None) == -1 and act(gz=None, gb=None) == -1 and act(ldz=7) == -1
    assert act(ws=None) == -3 and act(dt=3) == -4 and act(a=9) == -1
    dg = lambda gz=ONE, ldg=8, ldw=64, dt=BF16: lib.gnn_linear_dgrad(gz, ldg, ONE, ldw, dt, ONE, 4, 8, 64, None, 0, ONE, None)
    wg = lambda gz=ONE, ldg=8, ldx=64, dt=BF16: lib.gnn_linear_wgrad(gz, ldg, ONE, ldx, dt, ONE, 4, 8, 64, None, 0, ONE, None)
    for f in (dg, wg):
        assert f(gz=None) == -1 and f(ldg=7) == -1 and f(ldg=12) == -4 and f(dt=3) == -4
        assert f(dt=F32) == -3 and f(dt=F32, ldg=12) == -4


def test_linear_bwd_c_refusals():
    from ae_mlsys_gnn_b200 import _capi

    lib = _capi.lib()
    need = ctypes.c_size_t(0)
    size = lambda M=100, N=64, dt=1, own=1: lib.gnn_linear_bwd_workspace_bytes(M, N, 64, dt, own, ctypes.byref(need))
    assert size() == 0 and need.value >= 100 * 64 * 2
    assert size(N=0) == -1 and size(M=-1) == -1 and size(dt=3) == -1 and size() == 0
    bwd = lambda act=4, own=1, ws=ONE, nb=need.value, dt=1, M=100: lib.gnn_linear_bwd(
        ONE, ONE, act, 0.2, ONE, 64, ONE, 64, dt, own, ONE, ONE, ONE, M, 64, 64, ws, nb, ONE, None)
    assert bwd(own=0) == -1 and bwd(ws=None) == -3 and bwd(nb=need.value - 1) == -3
    assert bwd(dt=3) == -4 and bwd(M=-1) == -1


def test_pad_rows_c_refusals():
    from ae_mlsys_gnn_b200 import _capi

    lib = _capi.lib()
    pad = lambda src=ONE, size=2, rows=4, cols=5, dst=ONE, ld=8: lib.gnn_pad_rows(src, size, rows, cols, dst, ld, None)
    assert pad(rows=0) == 0
    assert pad(src=None) == -1 and pad(dst=None) == -1 and pad(dst=ctypes.c_void_p(264)) == -1
    assert pad(src=ctypes.c_void_p(257)) == -1 and pad(ld=4) == -1 and pad(ld=12) == -1
    assert pad(size=8) == -4 and pad(rows=-1) == -1 and pad(cols=0) == -1


def test_linear_refuses_cpu_tensors():
    from ae_mlsys_gnn_b200.operators.linear_act import linear_act, linear_act_fp8

    with pytest.raises(ValueError, match="CUDA"):
        linear_act(torch.zeros(2, 8), torch.zeros(4, 8))
    with pytest.raises(TypeError):
        linear_act([0.0], torch.zeros(4, 8))
    with pytest.raises(ValueError, match="CUDA"):
        linear_act_fp8(torch.zeros(2, 8).to(torch.float8_e4m3fn), torch.ones(2), torch.zeros(4, 8).to(torch.float8_e4m3fn),
                       torch.ones(4))
