"""Rows between token order and expert order, for layers whose rows choose k of E experts (no
counterpart in the reference; the neighbours here are csr2csc, the stable sort of edges by column,
and mhspmm, the weighted sum of rows).

    order = expert_sort(ids, E)              # ids (T, k): the experts every token chose
    xs = expert_dispatch(x, order)           # (T*k, D): the tokens' rows, expert after expert
    ...                                      # expert e works on rows offsets[e] .. offsets[e+1]
    out = expert_combine(ys, weights, order) # out[t] = sum_j weights[t, j] * ys[slots[t, j]]

The sort is stable and exact; nothing is read back to the host.  A pair whose id is not one of
0..E-1 (a padding token's -1) goes nowhere and adds nothing.  Rows are float32, bfloat16 or float16;
sums are fp32 in the order of the choices, each result is rounded once, no atomics are used.
"""
from __future__ import annotations

import torch

from .. import _capi as capi

I32 = torch.int32


class ExpertOrder:
    """What ``expert_sort`` found: ``offsets`` (E+1) int32, the first row of every expert and the
    number of rows in use; ``slots`` (T, k) int32, the row of every (token, choice) pair or -1."""

    __slots__ = ("offsets", "slots", "n_experts", "tokens", "k", "_kept")

    def __init__(self, offsets, slots, n_experts):
        self.offsets, self.slots, self.n_experts = offsets, slots, n_experts
        self.tokens, self.k = slots.shape
        self._kept = offsets.data_ptr() + 4 * n_experts  # device address of the number of rows in use


def expert_sort(ids, n_experts: int) -> ExpertOrder:
    """Stable counting sort of the (token, choice) pairs of ``ids`` (T, k), int32 or int64, by expert.
    At most 1024 experts and 32 choices."""
    if not isinstance(ids, torch.Tensor):
        raise TypeError("ids must be a torch.Tensor")
    if not ids.is_cuda:
        raise ValueError("ids must be a CUDA tensor (no CPU path exists)")
    if ids.dtype not in (torch.int32, torch.int64):
        raise TypeError(f"ids must be int32 or int64, got {ids.dtype}")
    if ids.dim() != 2 or not 1 <= ids.shape[1] <= 32:
        raise ValueError(f"ids must be (tokens, choices) with 1 to 32 choices, got shape {tuple(ids.shape)}")
    if not 1 <= n_experts <= 1024:
        raise ValueError(f"n_experts must be 1 to 1024, got {n_experts}")
    ids = ids if ids.is_contiguous() else ids.contiguous()
    dev = ids.device
    slots = torch.empty(ids.shape, dtype=I32, device=dev)
    offsets = torch.empty(n_experts + 1, dtype=I32, device=dev)
    pairs = ids.numel()
    ws, nbytes = capi.scratch("gnn_expert_sort_workspace_bytes", dev, pairs, n_experts)
    capi.launch(dev, "gnn_expert_sort", ids.data_ptr(), int(ids.dtype is torch.int64), pairs, n_experts,
                offsets.data_ptr(), slots.data_ptr(), capi.ptr(ws), nbytes)
    return ExpertOrder(offsets, slots, n_experts)


def _check_order(order, dev):
    if not isinstance(order, ExpertOrder):
        raise TypeError("order must come from expert_sort")
    if order.slots.device != dev:
        raise ValueError(f"order is on {order.slots.device}, expected {dev}")


def _dispatch(x, order):
    d = x.shape[1]
    out = torch.empty((order.tokens * order.k, d), dtype=x.dtype, device=x.device)
    if d:
        capi.launch(x.device, "gnn_expert_dispatch", x.data_ptr(), order.slots.data_ptr(), order._kept,
                    capi.DTYPE_CODES[x.dtype], order.tokens, order.k, d, out.data_ptr())
    return out


def _combine(rows, weights, order):
    d = rows.shape[1]
    out = torch.empty((order.tokens, d), dtype=rows.dtype, device=rows.device)
    if d:
        wdt = rows.dtype if weights is None else weights.dtype
        capi.launch(rows.device, "gnn_expert_combine", rows.data_ptr(), capi.ptr(weights), order.slots.data_ptr(),
                    capi.DTYPE_CODES[rows.dtype], capi.DTYPE_CODES[wdt], order.tokens, order.k, d, out.data_ptr())
    return out


class _Dispatch(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, order):
        ctx.order = order
        return _dispatch(x, order)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, g):
        return _combine(g.contiguous(), None, ctx.order), None


class _Combine(torch.autograd.Function):
    @staticmethod
    def forward(ctx, rows, weights, order):
        ctx.save_for_backward(rows, weights)
        ctx.order = order
        return _combine(rows, weights, order)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, g):
        rows, weights = ctx.saved_tensors
        order, g = ctx.order, g.contiguous()
        d = rows.shape[1]
        g_rows = torch.empty_like(rows)
        if not d:
            return g_rows, torch.zeros_like(weights), None
        g_weights = torch.empty_like(weights) if ctx.needs_input_grad[1] else None
        capi.launch(rows.device, "gnn_expert_combine_bwd", g.data_ptr(), rows.data_ptr(), weights.data_ptr(),
                    order.slots.data_ptr(), order._kept, capi.DTYPE_CODES[rows.dtype], capi.DTYPE_CODES[weights.dtype],
                    order.tokens, order.k, d, g_rows.data_ptr(), capi.ptr(g_weights))
        return g_rows, g_weights, None


def expert_dispatch(x, order: ExpertOrder):
    """Rows of x (T, D) in expert order: (T*k, D), row slots[t, j] = x[t]; the rows behind the last
    one in use are zero.  Differentiable: grad_x[t] is the sum of its rows' gradients."""
    x = capi.rows_of(x, "x")
    _check_order(order, x.device)
    if x.dim() != 2 or x.shape[0] != order.tokens:
        raise ValueError(f"x must be ({order.tokens}, D), got {tuple(x.shape)}")
    if capi.recorded(x):
        return _Dispatch.apply(x, order)
    return _dispatch(x, order)


def expert_combine(rows, weights, order: ExpertOrder):
    """out[t] = sum_j weights[t, j] * rows[slots[t, j]] for rows (T*k, D) in expert order and weights
    (T, k) of the rows' type or float32.  Differentiable in rows and weights."""
    rows = capi.rows_of(rows, "rows")
    _check_order(order, rows.device)
    if rows.dim() != 2 or rows.shape[0] != order.tokens * order.k:
        raise ValueError(f"rows must be ({order.tokens * order.k}, D), got {tuple(rows.shape)}")
    weights = capi.rows_of(weights, "weights")
    if weights.dtype not in (rows.dtype, torch.float32):
        raise TypeError(f"weights must be {rows.dtype} or float32, got {weights.dtype}")
    if weights.device != rows.device:
        raise ValueError(f"weights is on {weights.device}, expected {rows.device}")
    if weights.shape != order.slots.shape:
        raise ValueError(f"weights must be {tuple(order.slots.shape)}, got {tuple(weights.shape)}")
    if capi.recorded(rows, weights):
        return _Combine.apply(rows, weights, order)
    return _combine(rows, weights, order)
