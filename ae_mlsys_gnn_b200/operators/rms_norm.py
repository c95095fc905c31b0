"""Root-mean-square norm with the residual's addition (no counterpart in the reference, whose models
have no norm between their layers: script/train/train_gatconv_our.py:47-53).

    h = x + residual        y = h / sqrt(mean(h^2) + eps) * weight

``add_rms_norm`` returns y and the new residual stream h and is differentiable; ``add_rms_norm_fp8``
returns y as e4m3 values with fp32 scales, the form ``linear_act_fp8`` reads.  Rows are float32,
bfloat16 or float16, at most 32768 wide, with any leading dimensions; sums are fp32 whatever the
type, y is formed from the unrounded fp32 h, and every result is rounded once.
"""
from __future__ import annotations

import torch

from .. import _capi as capi

FP8 = torch.float8_e4m3fn


def _check(x, weight, residual):
    x = capi.rows_of(x, "x")
    d = x.shape[-1]
    if d < 1:
        raise ValueError("x must have at least one column")
    if isinstance(weight, torch.Tensor) and weight.dtype is torch.float32:
        weight = capi.rows_of(weight, "weight")
        if weight.device != x.device:
            raise ValueError(f"weight is on {weight.device}, expected {x.device}")
    else:
        weight = capi.rows_of(weight, "weight", x)
    if weight.dim() != 1 or weight.shape[0] != d:
        raise ValueError(f"weight must be a vector of {d} elements, got shape {tuple(weight.shape)}")
    if residual is not None:
        residual = capi.rows_of(residual, "residual", x)
        if residual.shape != x.shape:
            raise ValueError(f"residual must have x's shape {tuple(x.shape)}, got {tuple(residual.shape)}")
    return x, weight, residual, d


def _forward(x, weight, residual, eps, d, with_rstd):
    dev, n = x.device, x.numel() // d
    y = torch.empty_like(x)
    h = torch.empty_like(x) if residual is not None else None
    rstd = torch.empty(n, dtype=torch.float32, device=dev) if with_rstd else None
    code = capi.DTYPE_CODES
    capi.launch(dev, "gnn_rms_norm_fwd", x.data_ptr(), None if residual is None else residual.data_ptr(),
                weight.data_ptr(), code[x.dtype], code[weight.dtype], n, d, eps, y.data_ptr(),
                None if h is None else h.data_ptr(), None if rstd is None else rstd.data_ptr())
    return y, h, rstd


class _AddRmsNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, residual, eps):
        ctx.set_materialize_grads(False)
        y, h, rstd = _forward(x, weight, residual, eps, x.shape[-1], True)
        ctx.save_for_backward(x if h is None else h, weight, rstd)
        ctx.has_residual = h is not None
        return (y, h) if h is not None else y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, gy, gh=None):
        h, weight, rstd = ctx.saved_tensors
        if gy is None:  # only h was used
            return gh, None, (gh if ctx.has_residual else None), None
        d = h.shape[-1]
        n = h.numel() // d
        gy = gy.contiguous()
        gh = None if gh is None else gh.contiguous()
        gx = torch.empty_like(h)
        gw = ws = None
        nbytes = 0
        if ctx.needs_input_grad[1]:
            gw = torch.empty_like(weight)
            ws, nbytes = capi.scratch("gnn_rms_norm_bwd_workspace_bytes", h.device, n, d)
        capi.launch(h.device, "gnn_rms_norm_bwd", gy.data_ptr(), capi.ptr(gh), h.data_ptr(), weight.data_ptr(),
                    rstd.data_ptr(), capi.DTYPE_CODES[h.dtype], capi.DTYPE_CODES[weight.dtype], n, d, gx.data_ptr(),
                    capi.ptr(gw), capi.ptr(ws), nbytes)
        return gx, gw, (gx if ctx.has_residual else None), None


def add_rms_norm(x, weight, residual=None, eps: float = 1e-6):
    """(y, h) for x (..., D), weight (D,) of x's type or float32, residual of x's shape or None
    (then h is x itself).  Differentiable in x, weight and residual."""
    x, weight, residual, d = _check(x, weight, residual)
    if capi.recorded(x, weight, residual):
        out = _AddRmsNorm.apply(x, weight, residual, float(eps))
        return out if residual is not None else (out, x)
    y, h, _ = _forward(x, weight, residual, eps, d, False)
    return y, (x if h is None else h)


def add_rms_norm_fp8(x, weight, residual=None, eps: float = 1e-6, block: int = 0):
    """(q, scale, h): y of ``add_rms_norm`` as ``torch.float8_e4m3fn`` values q with
    y ~ q * scale, scale = max(max|y| / 448, 2^-126) over a row (``block`` 0, scale (..., 1)) or over
    every 128 columns (``block`` 128, scale (..., ceil(D / 128))).  For inference: inputs that
    require a gradient are refused while gradients are recorded."""
    x, weight, residual, d = _check(x, weight, residual)
    if block not in (0, 128):
        raise ValueError("block must be 0 (one scale a row) or 128")
    if capi.recorded(x, weight, residual):
        raise RuntimeError("add_rms_norm_fp8 has no gradient: call it under torch.no_grad()")
    dev, n = x.device, x.numel() // d
    q = torch.empty_like(x, dtype=FP8)
    scale = torch.empty((*x.shape[:-1], -(-d // block) if block else 1), dtype=torch.float32, device=dev)
    h = torch.empty_like(x) if residual is not None else None
    code = capi.DTYPE_CODES
    capi.launch(dev, "gnn_rms_norm_fp8", x.data_ptr(), None if residual is None else residual.data_ptr(),
                weight.data_ptr(), code[x.dtype], code[weight.dtype], n, d, eps, block, q.data_ptr(), scale.data_ptr(),
                None if h is None else h.data_ptr())
    return q, scale, (x if h is None else h)
