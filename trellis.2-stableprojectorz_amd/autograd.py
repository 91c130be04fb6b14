"""Gradients of the differentiable ops (torch.autograd.Function around two C-ABI calls each).

The backward calls run on the stream that is current there, which is the forward's; their scratch
comes from torch's allocator, so a training step can be captured into a graph.
"""
from __future__ import annotations

import torch
from torch.autograd.function import once_differentiable

from . import ops


class GroupNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, cu, b, groups, eps, silu):
        stats = torch.empty((b, groups, 2), dtype=torch.float32, device=x.device)
        out = ops._group_norm(x, weight, bias, cu, b, groups, eps, silu, None, stats)
        ctx.save_for_backward(x, weight, bias, cu, stats)
        ctx.args = (b, groups, silu)
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x, weight, bias, cu, stats = ctx.saved_tensors
        b, groups, silu = ctx.args
        dx, dw, db = ops._group_norm_backward(dy.contiguous(), x, weight, bias, cu, b, groups, silu,
                                              stats, any(ctx.needs_input_grad[1:3]))
        return dx, dw, db, None, None, None, None, None


class DiffAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, lam, cq, ck, b, scale, max_q, max_kv):
        out, maps, lse = ops._diff_attention(q, k, v, lam, cq, ck, b, scale, max_q, max_kv, None, True)
        ctx.save_for_backward(q, k, v, lam, maps, lse, cq, ck)
        ctx.args = (b, scale, max_q, max_kv)
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, do):
        q, k, v, lam, maps, lse, cq, ck = ctx.saved_tensors
        do = do.contiguous()
        if do.data_ptr() % 16:  # a view into a larger gradient
            do = do.clone()
        grads = ops._diff_attention_backward(do, q, k, v, lam, maps, lse, cq, ck,
                                             *ctx.args)
        return (*grads, None, None, None, None, None, None)
