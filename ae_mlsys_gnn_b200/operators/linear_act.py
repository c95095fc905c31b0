"""Linear layer with bias, activation and residual in the product's epilogue (no counterpart module in
the reference, which composes nn.Linear, F.elu / F.leaky_relu and additions: layers/gmmconv_layer.py:68-75,
script/train/train_edgeconv_our.py:44-56).  ``dense.linear`` is the plain fp32 product beside it.

    z = x W^T + bias        y = act(z) + residual

``linear_act`` takes float32 (error-compensated 3xTF32, fp32-level accuracy), bfloat16 or float16 and
is differentiable; ``linear_act_fp8`` takes e4m3 operands with a scale for every row of x and of W
(what ``add_rms_norm_fp8`` makes).  Sums, bias, activation and residual are fp32, rounded once; the
gradient of z is rounded to the operands' type before its two products, and z itself is kept for the
backward pass in that type (a gradient at the rounded z: within the rounding of the result).

Error contract as in ``dense``: every wait inside the product kernels is bounded; ``dense.check_status()``
reads the status word (a device synchronisation) and raises if one expired.
"""
from __future__ import annotations

import torch

from .. import _capi as capi
from . import dense

FP8 = torch.float8_e4m3fn
E4M3_CODE = 3
ACTIVATIONS = {None: 0, "relu": 1, "leaky_relu": 2, "elu": 3, "gelu": 4, "silu": 5}


def _status(dev):
    """The device's status word; it has to outlive every graph, so it is not made while one is captured."""
    t = dense._status.get(dev.index)
    if t is None:
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError("the first matrix product on a device must run before a graph is captured")
        with torch.inference_mode(False):  # it is also reset outside of inference mode
            t = dense._status_word(dev)
    return t


def _operand(t):
    """(tensor, row pitch in elements) of a contiguous matrix as the product kernels read it: rows a
    multiple of 16 bytes apart that start on a 16-byte boundary; others are copied to such a pitch, with
    zeros behind the columns (in fp32 the reduction runs over them)."""
    k, size = t.shape[1], t.element_size()
    per = 16 // size
    if k % per == 0:
        return (t if t.data_ptr() % 16 == 0 else t.clone()), k
    ld = -(-k // per) * per
    buf = torch.empty((t.shape[0], ld), dtype=t.dtype, device=t.device)
    capi.launch(t.device, "gnn_pad_rows", t.data_ptr(), size, t.shape[0], k, buf.data_ptr(), ld)
    return buf, ld


def _forward(x, xs, weight, ws, bias, act, residual, slope, out_dtype, want_z):
    """x (M, K) and weight (N, K) as the kernels read them -> (y, z or None).  K is the logical width."""
    (x, ldx, K), (weight, ldw) = x, weight
    dev = x.device
    M, N = x.shape[0], weight.shape[0]
    y = torch.empty((M, N), dtype=out_dtype, device=dev)
    z = torch.empty((M, N), dtype=out_dtype, device=dev) if want_z else None
    code = capi.DTYPE_CODES.get(x.dtype, E4M3_CODE)
    if code == 0:
        K = ldx  # zero columns behind the last
    if M and N:
        scratch, nbytes = capi.scratch("gnn_linear_fwd_workspace_bytes", dev, M, N, K, code)
        ptr = capi.ptr
        capi.launch(dev, "gnn_linear_fwd", x.data_ptr(), ldx, weight.data_ptr(), ldw, code, ptr(xs), ptr(ws), ptr(bias), act,
                    slope, ptr(residual), y.data_ptr(), ptr(z), capi.DTYPE_CODES[out_dtype], M, N, K, ptr(scratch), nbytes,
                    _status(dev).data_ptr())
    return y, z


class _LinearAct(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, residual, act, slope):
        xo, ldx = _operand(x)
        wo, ldw = _operand(weight)
        # bias and activation share their pass of the backward; without an activation z is not needed
        need_z = act != 0 and any(ctx.needs_input_grad[:3])
        y, z = _forward((xo, ldx, x.shape[1]), None, (wo, ldw), None, bias, act, residual, slope, x.dtype, need_z)
        # the fp32 products take any row pitch of the weights, the others read them by TMA
        ctx.save_for_backward(xo, weight if x.dtype is torch.float32 else wo, z)
        ctx.args = (x.shape, act, slope)
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, gy):
        x, w, z = ctx.saved_tensors
        (M, K), act, slope = ctx.args
        N, dt, dev = w.shape[0], x.dtype, x.device
        code = capi.DTYPE_CODES[dt]
        need_x, need_w, need_b, need_r = ctx.needs_input_grad[:4]
        gy = gy.contiguous()
        gx = gw = gb = None
        per = 16 // x.element_size()
        ldz = -(-N // per) * per
        products = (need_x or need_w) and M > 0
        if products and (code != 0 or (N % 4 == 0 and K % 4 == 0)):  # one call for all steps
            own = int(act != 0 or ldz != N or gy.data_ptr() % 16 != 0)
            gx = torch.empty((M, K), dtype=dt, device=dev) if need_x else None
            gw = torch.empty((N, K), dtype=dt, device=dev) if need_w else None
            gb = torch.empty(N, dtype=dt, device=dev) if need_b else None
            scratch, nbytes = capi.scratch("gnn_linear_bwd_workspace_bytes", dev, M, N, K, code, own)
            ptr = capi.ptr
            capi.launch(dev, "gnn_linear_bwd", gy.data_ptr(), ptr(z), act, slope, x.data_ptr(), x.shape[1], w.data_ptr(),
                        w.shape[1], code, own, ptr(gx), ptr(gw), ptr(gb), M, N, K, scratch.data_ptr(), nbytes,
                        _status(dev).data_ptr())
            return gx, gw, gb, (gy if need_r else None), None, None
        gz = gy
        own_gz = products and (act != 0 or ldz != N or gy.data_ptr() % 16 != 0)
        if own_gz:
            gz = torch.empty((M, ldz), dtype=dt, device=dev)
        if need_b:
            gb = torch.empty(N, dtype=dt, device=dev)
        if own_gz or need_b:
            scratch, nbytes = capi.scratch("gnn_linear_act_bwd_workspace_bytes", dev, M, N, ldz) if need_b else (None, 0)
            capi.launch(dev, "gnn_linear_act_bwd", gy.data_ptr(), capi.ptr(z), act, slope, code, M, N,
                        gz.data_ptr() if own_gz else None, ldz, capi.ptr(gb), capi.ptr(scratch), nbytes)
        if need_x:
            gx = torch.empty((M, K), dtype=dt, device=dev)
            if M:
                wr, n = w, N
                if code == 0 and ldz != N:  # the reduction runs over the zero columns of gz
                    wr, n = torch.nn.functional.pad(w, (0, 0, 0, ldz - N)), ldz
                scratch, nbytes = capi.scratch("gnn_linear_dgrad_workspace_bytes", dev, M, n, K, code)
                capi.launch(dev, "gnn_linear_dgrad", gz.data_ptr(), ldz, wr.data_ptr(), wr.shape[1], code, gx.data_ptr(),
                            M, n, K, capi.ptr(scratch), nbytes, _status(dev).data_ptr())
        if need_w:
            gw = torch.empty((N, K), dtype=dt, device=dev)
            n, k, out = N, K, gw
            if code == 0:
                n, k = ldz, x.shape[1]
                if n != N or k != K:
                    out = torch.empty((n, k), dtype=dt, device=dev)
            scratch, nbytes = capi.scratch("gnn_linear_wgrad_workspace_bytes", dev, M, n, k, code)
            capi.launch(dev, "gnn_linear_wgrad", gz.data_ptr(), ldz, x.data_ptr(), x.shape[1], code, out.data_ptr(), M, n,
                        k, capi.ptr(scratch), nbytes, _status(dev).data_ptr())
            if out is not gw:
                gw.copy_(out[:N, :K])
        return gx, gw, gb, (gy if need_r else None), None, None


def _check_epilogue(lead, N, dtype, dev, bias, activation, residual):
    if activation not in ACTIVATIONS:
        raise ValueError(f"activation must be one of {list(ACTIVATIONS)}, got {activation!r}")
    for t, name, shape in ((bias, "bias", (N,)), (residual, "residual", (*lead, N))):
        if t is None:
            continue
        if not isinstance(t, torch.Tensor):
            raise TypeError(f"{name} must be a torch.Tensor")
        if not t.is_cuda or t.device != dev:
            raise ValueError(f"{name} must be on {dev}, got {t.device}")
        if t.dtype != dtype:
            raise TypeError(f"{name} must be {dtype}, got {t.dtype}")
        if t.shape != shape:
            raise ValueError(f"{name} must have shape {shape}, got {tuple(t.shape)}")


def linear_act(x, weight, bias=None, activation=None, residual=None, negative_slope: float = 0.2):
    """act(x W^T + bias) + residual for x (..., K), weight (N, K), bias (N,) and residual (..., N), all of
    one type: float32, bfloat16 or float16.  ``activation``: None, "relu", "leaky_relu" (with
    ``negative_slope``), "elu", "gelu" (the erf form) or "silu".  Differentiable in all four tensors."""
    x = capi.rows_of(x, "x")
    weight = capi.rows_of(weight, "weight", x)
    if weight.dim() != 2 or weight.shape[1] != x.shape[-1]:
        raise ValueError(f"weight must be (N, {x.shape[-1]}), got {tuple(weight.shape)}")
    if x.shape[-1] < 1 or weight.shape[0] < 1:
        raise ValueError("x must have at least one column and weight at least one row")
    lead, N = x.shape[:-1], weight.shape[0]
    _check_epilogue(lead, N, x.dtype, x.device, bias, activation, residual)
    act, slope = ACTIVATIONS[activation], float(negative_slope)
    x2 = x if x.dim() == 2 else x.reshape(-1, x.shape[-1])
    if residual is not None:
        residual = residual.contiguous()
        if residual.dim() != 2:
            residual = residual.view(-1, N)
    if bias is not None:
        bias = bias.contiguous()
    if capi.recorded(x2, weight, bias, residual):
        y = _LinearAct.apply(x2, weight, bias, residual, act, slope)
    else:
        y, _ = _forward((*_operand(x2), x2.shape[1]), None, _operand(weight), None, bias, act, residual, slope, x.dtype,
                        False)
    return y if x.dim() == 2 else y.view(*lead, N)


def _scale_of(t, name, rows, dev):
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor")
    if not t.is_cuda or t.device != dev:
        raise ValueError(f"{name} must be on {dev}, got {t.device}")
    if t.dtype != torch.float32:
        raise TypeError(f"{name} must be float32, got {t.dtype}")
    if t.numel() != rows:
        raise ValueError(f"{name} must hold one scale a row ({rows}), got shape {tuple(t.shape)}")
    return t.contiguous()


def linear_act_fp8(x8, x_scale, weight8, weight_scale, bias=None, activation=None, residual=None,
                   negative_slope: float = 0.2, out_dtype: torch.dtype = torch.bfloat16):
    """``linear_act`` on ``torch.float8_e4m3fn`` operands: x ~ x8 (..., K) * x_scale (one per row),
    W ~ weight8 (N, K) * weight_scale (one per row).  bias, residual and the result are ``out_dtype``
    (float32, bfloat16 or float16).  For inference: there is no gradient, and operands of the epilogue
    that require one are refused while gradients are recorded."""
    for t, name in ((x8, "x8"), (weight8, "weight8")):
        if not isinstance(t, torch.Tensor):
            raise TypeError(f"{name} must be a torch.Tensor")
        if not t.is_cuda:
            raise ValueError(f"{name} must be a CUDA tensor (no CPU path exists)")
        if t.dtype != FP8:
            raise TypeError(f"{name} must be float8_e4m3fn, got {t.dtype}")
    dev = x8.device
    if weight8.device != dev:
        raise ValueError(f"weight8 is on {weight8.device}, expected {dev}")
    if x8.dim() < 1 or weight8.dim() != 2 or weight8.shape[1] != x8.shape[-1] or weight8.numel() < 1:
        raise ValueError(f"x8 must be (..., K) and weight8 (N, K), got {tuple(x8.shape)} and {tuple(weight8.shape)}")
    if out_dtype not in capi.DTYPE_CODES:
        raise TypeError(f"out_dtype must be float32, bfloat16 or float16, got {out_dtype}")
    lead, N, K = x8.shape[:-1], weight8.shape[0], x8.shape[-1]
    _check_epilogue(lead, N, out_dtype, dev, bias, activation, residual)
    x2 = x8.contiguous()
    if x2.dim() != 2:
        x2 = x2.view(-1, K)
    xs = _scale_of(x_scale, "x_scale", x2.shape[0], dev)
    ws = _scale_of(weight_scale, "weight_scale", N, dev)
    if capi.recorded(xs, ws, bias, residual):
        raise RuntimeError("linear_act_fp8 has no gradient: call it under torch.no_grad()")
    if bias is not None:
        bias = bias.contiguous()
    if residual is not None:
        residual = residual.contiguous()
    xo, ldx = _operand(x2)
    y, _ = _forward((xo, ldx, K), xs, _operand(weight8.contiguous()), ws, bias, ACTIVATIONS[activation], residual,
                    float(negative_slope), out_dtype, False)
    return y if x8.dim() == 2 else y.view(*lead, N)
