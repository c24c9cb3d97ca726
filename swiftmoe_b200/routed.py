"""The routed rows as differentiable operators: tokens sorted by expert, the experts'
linear layers, and the rows back in token order.

    rows, plan = sort_tokens(x, idx, num_experts)               # idx from kernels.router
    h = grouped_linear(rows, w_in, plan["offsets"], bias=b_in, activation="gelu")
    y = grouped_linear(h, w_out, plan["offsets"], bias=b_out)
    out = unsort_tokens(y, plan, weights=w, residual=x)

The layers (``StandardMoE`` / ``UltimateMoE``) run their own bias-free linear or SwiGLU
experts in one call; these are the pieces for experts of another kind, with gradients.  No
call waits for the device, and all of them can be captured into a CUDA graph, forward and
backward.  (A backward captured while an eager graph of the same leaf tensors is alive
accumulates into leaves whose stream torch recorded outside the capture, which torch does
not allow; drop the eager graph's outputs before capturing, or call the ``kernels``
functions that the backward consists of.)

Reverse mode only: a tensor with a forward-mode tangent is refused, and so is a second
derivative.

The reference's pieces are forward-only: models/ultimate_moe.py:118-125 (dispatch), 145-155
(combine), 237-250 and models/baseline_moe.py:151-162 (experts).
"""
from __future__ import annotations

from typing import Optional, Tuple

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from . import _lib as L
from . import kernels as K


def _grads_wanted(*ts) -> bool:
    # Tangents are refused here: the kernels read memory, where a dual tensor's is not, and
    # such tensors need not have requires_grad set.  (_current_level: -1 outside a dual level)
    if forward_ad._current_level >= 0 and any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in ts):
        raise L.SwiftMoEError("forward-mode derivatives of the routed rows are not supported")
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in ts)


def _sizes(plan: dict) -> dict:
    """What a backward needs of a plan besides tensors, as it is now: the dict is the caller's."""
    return {"T": plan["T"], "k": plan["k"], "rows_cap": plan["rows_cap"], "row_align": plan.get("row_align")}


class _SortTokens(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w, args, made):
        rows, plan = K.sort_tokens(x, args[0], args[1], w, args[2], args[3])
        made.append(plan)
        ctx.sizes = _sizes(plan)
        ctx.save_for_backward(x if ctx.needs_input_grad[1] else None, w, plan["slot_row"])
        return rows

    @staticmethod
    @once_differentiable
    def backward(ctx, drows):
        x, w, slot_row = ctx.saved_tensors
        drows, plan = drows.contiguous(), dict(ctx.sizes, slot_row=slot_row)
        need_x, need_w = ctx.needs_input_grad[:2]
        if need_w and not need_x:
            return None, K.sort_rows(x, plan, w, rows_cap=drows.shape[0], y=drows, only_dw=True), None, None
        if need_w:
            return *K.unsort_rows(drows, plan, w, x=x), None, None
        return K.unsort_rows(drows, plan, w), None, None, None


class _UnsortTokens(torch.autograd.Function):
    @staticmethod
    def forward(ctx, rows, w, residual, plan):
        ctx.sizes, ctx.rows_cap = _sizes(plan), rows.shape[0]
        need_rows, need_w = ctx.needs_input_grad[:2]
        ctx.save_for_backward(rows if need_w else None, w, plan["slot_row"], plan["offsets"] if need_rows else None,
                              plan["row_token"] if need_rows and plan.get("row_align") != 1 else None)
        return K.unsort_rows(rows, plan, w, residual)

    @staticmethod
    @once_differentiable
    def backward(ctx, dout):
        rows, w, slot_row, offsets, row_token = ctx.saved_tensors
        need_rows, need_w, need_res, _ = ctx.needs_input_grad
        dout, plan = dout.contiguous(), dict(ctx.sizes, slot_row=slot_row, offsets=offsets, row_token=row_token)
        drows = dw = None
        if need_w and not need_rows:
            dw = K.sort_rows(dout, plan, w, rows_cap=ctx.rows_cap, y=rows, only_dw=True)
        elif need_w:
            drows, dw = K.sort_rows(dout, plan, w, rows_cap=ctx.rows_cap, y=rows)
        elif need_rows:
            drows = K.sort_rows(dout, plan, w, rows_cap=ctx.rows_cap)
        return drows, dw, dout if need_res else None, None


class _GroupedLinear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, a, weight, bias, residual, offsets, activation):
        need_a, need_w, need_b, _ = ctx.needs_input_grad[:4]
        keep = activation != "none" and (need_a or need_w or need_b)
        if a.dim() != 2 or weight.dim() != 3:
            raise L.SwiftMoEError("a must be [rows, K], weight [G, N, K]")
        z = torch.empty((a.shape[0], weight.shape[1]), dtype=a.dtype, device=a.device) if keep else None
        out = K.grouped_linear(a, weight, offsets, bias, activation, residual, preact=z)
        ctx.activation, ctx.bias_dtype = activation, bias.dtype if need_b else None
        ctx.save_for_backward(a if need_w else None, weight if need_a else None, offsets, z)
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, dout):
        a, weight, offsets, z = ctx.saved_tensors
        need_a, need_w, need_b, need_res = ctx.needs_input_grad[:4]
        dout = dout.contiguous()
        if dout.data_ptr() % 16:   # a piece of a larger gradient: the kernels load 16 bytes at a time
            dout = dout.clone()
        da = dw = db = None
        if need_a or need_w:
            da, dw, db = K.grouped_linear_bwd(dout, a, weight, offsets, ctx.activation, z, need_a=need_a, need_w=need_w,
                                              bias_dtype=ctx.bias_dtype)
        elif need_b:
            _, db = K.linear_act_bwd(dout, offsets, ctx.activation, z, ctx.bias_dtype)
        return da, dw, db, dout if need_res else None, None, None


def sort_tokens(x: torch.Tensor, idx: torch.Tensor, num_experts: int, weights: Optional[torch.Tensor] = None, *,
                capacity: int = 0, row_align: int = 1) -> Tuple[torch.Tensor, dict]:
    """(rows [R, d], plan): the tokens' rows grouped by expert, in (token, slot) order inside
    an expert, and the dispatch plan (``kernels.dispatch_plan``; ``plan["offsets"]`` [E+1]
    are the experts' row ranges, ``plan["counts"]`` the rows routed to each).

    x [T, d] fp32 / fp16 / bf16; idx [T, k] int32 expert of every slot, -1 for none (k <=
    32); weights [T, k] fp32 multiplies the rows (default: rows are copies).  At most
    ``capacity`` rows per expert are kept (0: all), group starts are multiples of
    ``row_align``.  R is the plan's upper bound on the rows; rows of no slot are zero.
    Differentiable in x and weights."""
    if _grads_wanted(x, weights):
        made = []
        rows = _SortTokens.apply(x, weights, (idx, num_experts, capacity, row_align), made)
        return rows, made[0]
    return K.sort_tokens(x, idx, num_experts, weights, capacity, row_align)


def unsort_tokens(rows: torch.Tensor, plan: dict, weights: Optional[torch.Tensor] = None,
                  residual: Optional[torch.Tensor] = None) -> torch.Tensor:
    """out [T, d]: the rows of every token summed in slot order, each times its weight
    (``weights`` [T, k] fp32, default 1), plus ``residual`` [T, d].  Dropped slots add
    nothing.  fp32 sums, one rounding.  Differentiable in rows, weights and residual."""
    if _grads_wanted(rows, weights, residual):
        return _UnsortTokens.apply(rows, weights, residual, plan)
    return K.unsort_rows(rows, plan, weights, residual)


def grouped_linear(a: torch.Tensor, weight: torch.Tensor, offsets: torch.Tensor, bias: Optional[torch.Tensor] = None,
                   activation: str = "none", residual: Optional[torch.Tensor] = None) -> torch.Tensor:
    """out [R, N] = act(a W_g^T + bias[g]) + residual for the rows [offsets[g], offsets[g+1]) of
    every group g; rows of no group are the residual alone (zeros without one).

    a [R, K] and weight [G, N, K] bf16 / fp16, K and N multiples of 8; offsets [G+1] int32 on
    the device (``plan["offsets"]``; groups may start anywhere); bias [G, N] in a's dtype or
    fp32; activation "none", "relu", "gelu" (exact), "gelu_tanh" or "silu"; residual [R, N].
    fp32 accumulation, one rounding; an activation's own relative error is 2^-19, at |z| = 10 up
    to 2^-15 (that of an exponential's argument).  Differentiable in a, weight, bias and
    residual.  With an activation two things are rounded to a's dtype on the way back: the
    pre-activations that the forward keeps, and the gradient dz in front of them, which da
    and dweight are products of (dbias sums it unrounded)."""
    K._act_code(activation)
    if _grads_wanted(a, weight, bias, residual):
        return _GroupedLinear.apply(a, weight, bias, residual, offsets, activation)
    return K.grouped_linear(a, weight, offsets, bias, activation, residual)
