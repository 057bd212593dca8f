"""The text encoder's operators with autograd: the forward and backward entry points of `aether_amd.ops` as differentiable functions.

Each call outside of `torch.no_grad()` keeps what its backward pass needs (rms_norm: the sum, or with a bfloat16 stream both of its terms; relbias_attn: its output in two bf16 parts and the rows'
log-sums; gated_ff: both projections in fp32).  Gradients are first order, and the same bits every time.

Into a captured graph, record the backward pass with `torch.autograd.grad` on leaves that no eager graph holds at that time: `Tensor.backward` accumulates
into `.grad` on the stream the leaf was first used on, and that stream does not take part in the capture.
"""
from __future__ import annotations

import torch
from torch.autograd.function import once_differentiable

from . import ops


class _RmsNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, delta, w, eps):
        y, res = ops.rms_norm(x, w, eps, delta=delta)
        again = delta is not None and x.dtype == torch.bfloat16          # the stored sum is rounded, the norm's was not
        ctx.save_for_backward(x if again else res, w, delta if again else None)
        ctx.eps, ctx.summed = eps, delta is not None
        ctx.set_materialize_grads(False)
        return (y, res) if ctx.summed else y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy, dres=None):
        res, w, delta = ctx.saved_tensors
        need_x, need_delta, need_w = ctx.needs_input_grad[:3]
        if dy is None and dres is None:
            return None, None, None, None
        if dy is None:                      # only the sum was used
            return dres if need_x else None, dres.to(torch.bfloat16, copy=True) if need_delta else None, torch.zeros_like(w) if need_w else None, None
        dx, ddelta, dw = ops.rms_norm_backward(dy, res, w, ctx.eps, dres=dres, need_ddelta=need_delta, delta=delta)
        return dx if need_x else None, ddelta, dw if need_w else None, None


def rms_norm(x, w, eps=1e-6, delta=None):
    """`ops.rms_norm` with gradients for x, delta and w."""
    if delta is None:
        return _RmsNorm.apply(x, None, w, eps), x
    return _RmsNorm.apply(x, delta, w, eps)


class _RelbiasAttn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, table, max_distance, scale, key_mask):
        o, lse = ops.relbias_attn(q, k, v, table, max_distance, scale, key_mask, need_lse=True)
        ctx.save_for_backward(q, k, v, table, o, lse, key_mask)
        ctx.max_distance, ctx.scale = max_distance, scale
        return o

    @staticmethod
    @once_differentiable
    def backward(ctx, do):
        q, k, v, table, o, lse, key_mask = ctx.saved_tensors
        need = ctx.needs_input_grad
        dq, dk, dv, dtable = ops.relbias_attn_backward(do, q, k, v, o, lse, table, ctx.max_distance, ctx.scale, key_mask, need_dtable=need[3])
        return dq if need[0] else None, dk if need[1] else None, dv if need[2] else None, dtable, None, None, None


def relbias_attn(q, k, v, table, max_distance=128, scale=1.0, key_mask=None):
    """`ops.relbias_attn` with gradients for q, k, v and the table."""
    return _RelbiasAttn.apply(q, k, v, table, max_distance, scale, key_mask)


class _GatedFf(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, wg, wu, act):
        h, gu = ops.gated_ff(x, wg, wu, act, need_gu=True)
        ctx.save_for_backward(x, wg, wu, gu)
        ctx.act = act
        return h

    @staticmethod
    @once_differentiable
    def backward(ctx, dh):
        x, wg, wu, gu = ctx.saved_tensors
        need = ctx.needs_input_grad
        dx, dwg, dwu = ops.gated_ff_backward(dh, x, wg, wu, gu, ctx.act, need_dx=need[0], need_dw=need[1] or need[2])
        return dx, dwg if need[1] else None, dwu if need[2] else None, None


def gated_ff(x, wg, wu, act="gelu_tanh"):
    """`ops.gated_ff` with gradients for x, wg and wu.  More rows than the backward pass takes (rows · 2F of 2^31) are refused here; without gradients
    `ops.gated_ff` has no such limit."""
    return _GatedFf.apply(x, wg, wu, act)


def _turned(t):
    """tᵀ with its rows padded with zeros to a multiple of 64 (the inner dimension of `ops.gemm_bf16`)."""
    n = t.shape[0]
    out = t.new_zeros(t.shape[1], (n + 63) // 64 * 64) if n % 64 else t.new_empty(t.shape[1], n)
    out[:, :n] = t.t()
    return out


class _Linear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w):
        ctx.save_for_backward(x, w)
        return ops.gemm_bf16(x, w)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x, w = ctx.saved_tensors
        need = ctx.needs_input_grad
        dy = dy.contiguous()
        return ops.gemm_bf16(dy, _turned(w)) if need[0] else None, ops.gemm_bf16(_turned(dy), _turned(x)) if need[1] else None


def linear(x, w):
    """x wᵀ on `ops.gemm_bf16` (x bfloat16 [M, K], w bfloat16 [N, K], K a multiple of 64, N of 64) with gradients for both."""
    return _Linear.apply(x, w)
