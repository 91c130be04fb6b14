"""Gradients of the differentiable ops (torch.autograd.Function around two C-ABI calls each).

The backward calls run on the stream that is current there, which is the forward's; their scratch
comes from torch's allocator, so a training step can be captured into a graph.
"""
from __future__ import annotations

import torch
from torch.autograd.function import once_differentiable

from . import ops


def _save(ctx, *ts):
    """save_for_backward, and where the tensors are."""
    ctx.save_for_backward(*ts)
    ctx.places = [t if t is None else (t.data_ptr(), t.stride()) for t in ts]


def _saved(ctx):
    """(the saved tensors, whether a hook gave any of them back in another place or layout).  The gradients' C
    calls take what the forward call checked; the layouts of others have to be looked at again."""
    ts = ctx.saved_tensors
    return ts, [t if t is None else (t.data_ptr(), t.stride()) for t in ts] != ctx.places


class GroupNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, cu, b, groups, eps, silu):
        stats = torch.empty((b, groups, 2), dtype=torch.float32, device=x.device)
        out = ops._group_norm(x, weight, bias, cu, b, groups, eps, silu, None, stats)
        _save(ctx, x, weight, bias, cu, stats)
        ctx.args = (b, groups, silu)
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        (x, weight, bias, cu, stats), moved = _saved(ctx)
        b, groups, silu = ctx.args
        dx, dw, db = ops._group_norm_backward(dy.contiguous(), x, weight, bias, cu, b, groups, silu,
                                              stats, any(ctx.needs_input_grad[1:3]), moved)
        return dx, dw, db, None, None, None, None, None


class GatedNorm(torch.autograd.Function):
    """Takes (tensors, args, want_r, want_h) of ops._gated_norm, and of the tensors those that are there."""

    @staticmethod
    def forward(ctx, how, *given):
        tensors, args, want_r, want_h = how
        r, h, stats = ops._gated_norm(tensors, args, want_r, want_h, None, True)
        ctx.set_materialize_grads(False)
        _save(ctx, args[0], stats, *given)
        ctx.how = args[1:], [t is not None for t in tensors], want_r, want_h, () if stats is None else stats.shape
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
        (cu, stats, *given), moved = _saved(ctx)
        if not all(there):
            it, wanted = iter(given), iter(ctx.needs_input_grad[1:])
            given = [next(it) if t else None for t in there]
            wanted = [t and next(wanted) for t in there]
        else:
            wanted = ctx.needs_input_grad[1:]
        grads = ops._gated_norm_backward(given, (cu, *args), stats, dr, dh, wanted, stats_shape if moved else None)
        return (None, *[g for g, t in zip(grads, there) if t])


class DiffAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, lam, cq, ck, b, scale, max_q, max_kv):
        out, maps, lse = ops._diff_attention(q, k, v, lam, cq, ck, b, scale, max_q, max_kv, None, True)
        _save(ctx, q, k, v, lam, maps, lse, cq, ck)
        ctx.args = (k.shape[0], b, scale, max_q, max_kv)
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, do):
        (q, k, v, lam, maps, lse, cq, ck), moved = _saved(ctx)
        do = do.contiguous()
        if do.data_ptr() % 16:  # a view into a larger gradient
            do = do.clone()
        grads = ops._diff_attention_backward(do, q, k, v, lam, maps, lse, cq, ck, moved, *ctx.args)
        return (*grads, None, None, None, None, None, None)


class WindowAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, lds, args):
        out, lo, lse = ops._window_attention(q, k, v, lds, args, None, True)
        _save(ctx, q, k, v, out, lo, lse, *args[:2])
        ctx.args = args[2:], lds, k.shape
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, do):
        (q, k, v, out, lo, lse, cq, ck), moved = _saved(ctx)
        args, lds, kv_shape = ctx.args
        do = do.contiguous()
        if do.data_ptr() % 16:  # a view into a larger gradient
            do = do.clone()
        grads = ops._window_attention_backward(do, q, k, v, out, lo, lse, lds, kv_shape if moved else None,
                                               (cq, ck, *args))
        return (*grads, None, None)
