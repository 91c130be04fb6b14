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


class GatedNorm(torch.autograd.Function):
    """Takes (tensors, args, want_r, want_h) of ops._gated_norm, and of the tensors those that are there."""

    @staticmethod
    def forward(ctx, how, *given):
        tensors, args, want_r, want_h = how
        r, h, stats = ops._gated_norm(tensors, args, want_r, want_h, None, True)
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(args[0], stats, *given)
        ctx.how = args[1:], [t is not None for t in tensors], want_r, want_h, None if stats is None else stats.shape
        return (r, h) if want_r and want_h else r if want_r else h

    @staticmethod
    @once_differentiable
    def backward(ctx, *douts):
        args, there, want_r, want_h, stats_shape = ctx.how
        dr = douts[0] if want_r else None
        dh = douts[-1] if want_h else None
        if dr is None and dh is None:
            return (None,) * len(ctx.needs_input_grad)
        dr = None if dr is None else dr.contiguous()
        dh = None if dh is None else dh.contiguous()
        cu, stats, *given = ctx.saved_tensors
        if not all(there):
            it, wanted = iter(given), iter(ctx.needs_input_grad[1:])
            given = [next(it) if t else None for t in there]
            wanted = [t and next(wanted) for t in there]
        else:
            wanted = ctx.needs_input_grad[1:]
        grads = ops._gated_norm_backward(given, (cu, *args), stats, stats_shape, dr, dh, wanted)
        return (None, *[g for g, t in zip(grads, there) if t])


class DiffAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, lam, cq, ck, b, scale, max_q, max_kv):
        out, maps, lse = ops._diff_attention(q, k, v, lam, cq, ck, b, scale, max_q, max_kv, None, True)
        ctx.save_for_backward(q, k, v, lam, maps, lse, cq, ck)
        ctx.total_kv, ctx.args = k.shape[0], (b, scale, max_q, max_kv)
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, do):
        q, k, v, lam, maps, lse, cq, ck = ctx.saved_tensors
        do = do.contiguous()
        if do.data_ptr() % 16:  # a view into a larger gradient
            do = do.clone()
        grads = ops._diff_attention_backward(do, q, k, v, lam, maps, lse, ctx.total_kv, cq, ck,
                                             *ctx.args)
        return (*grads, None, None, None, None, None, None)


class WindowAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, lds, args):
        out, lo, lse = ops._window_attention(q, k, v, lds, args, None, True)
        ctx.save_for_backward(q, k, v, out, lo, lse, *args[:2])
        ctx.kv_shape, ctx.args = k.shape, args[2:]
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, do):
        q, k, v, out, lo, lse, cq, ck = ctx.saved_tensors
        do = do.contiguous()
        if do.data_ptr() % 16:  # a view into a larger gradient
            do = do.clone()
        grads = ops._window_attention_backward(do, q, k, v, out, lo, lse, ctx.kv_shape, (cq, ck, *ctx.args))
        return (*grads, None, None)
