"""Differentiable forms of the kernels, for fine-tuning a model with its sparse attention layers in place.

`sparse_attention` is `ops.sparse_attn_fwd` with `ops.sparse_attn_bwd` behind it, `qkv_prologue` likewise.  Both are single
nodes of the autograd graph; first derivatives only.  The mask and the work lists made from it are constants of the layer:
its selection is not differentiated.
"""
from __future__ import annotations

from typing import Optional

import torch
from torch.autograd.function import once_differentiable

from . import ops

__all__ = ["sparse_attention"]


class _SparseAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, lists, key_lists, limits, check_status):
        out, lse = ops.sparse_attn_fwd(q, k, v, lists.counts, lists.entries, order=lists.order, return_lse=True,
                                       check_status=check_status, **limits)
        ctx.save_for_backward(q, k, v, out, lse, lists.counts, lists.entries, lists.order, key_lists.counts,
                              key_lists.entries, key_lists.order)
        ctx.limits, ctx.check_status = limits, check_status
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, dout):
        q, k, v, out, lse, *lists = ctx.saved_tensors
        grads = ops.sparse_attn_bwd(dout.contiguous(), q, k, v, out, lse, ops.TileLists(*lists[:3]),
                                    ops.KeyLists(*lists[3:]), check_status=ctx.check_status, **ctx.limits)
        return tuple(g if need else None for g, need in zip(grads, ctx.needs_input_grad)) + (None,) * 4


def sparse_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, lists: ops.TileLists, key_lists: ops.KeyLists, *,
                     softmax_scale: Optional[float] = None, q_split: Optional[int] = None,
                     kv_len_lo: Optional[int] = None, kv_len_hi: Optional[int] = None,
                     check_status="deferred") -> torch.Tensor:
    """Block-sparse attention of (B, H, N, D) float16 or bfloat16 tensors, differentiable with respect to q, k and v.

    lists, key_lists: `ops.tile_lists` and `ops.key_lists` of the layer's mask; the other arguments are those of
    `ops.sparse_attn_fwd`.  Tensors that are not contiguous are copied.  What lies between the forward and the backward is
    q, k, v, the output and 4 bytes per row."""
    limits = dict(softmax_scale=softmax_scale, q_split=q_split, kv_len_lo=kv_len_lo, kv_len_hi=kv_len_hi)
    return _SparseAttention.apply(q.contiguous(), k.contiguous(), v.contiguous(), lists, key_lists, limits, check_status)
