"""Differentiable forms of the kernels, for fine-tuning a model with its sparse attention layers in place.

`sparse_attention` is `ops.sparse_attn_fwd` with `ops.sparse_attn_bwd` behind it, `qkv_prologue` likewise.  Both are single
nodes of the autograd graph; first derivatives only.  The mask and the work lists made from it are constants of the layer:
its selection is not differentiated.
"""
from __future__ import annotations

from typing import Optional, Tuple

import torch
from torch.autograd.function import once_differentiable

from . import _lib, ops

__all__ = ["sparse_attention", "qkv_prologue"]


def _builds_graph(*tensors: Optional[torch.Tensor]) -> bool:
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)


class _SparseAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, lists, key_lists, limits, check_status, return_lse, wanted):
        if check_status == "deferred" and q.is_cuda and not torch.cuda.is_current_stream_capturing():
            ops.check_posted_status(q.device)
        res = ops.sparse_attn_fwd(q, k, v, lists.counts, lists.entries, order=lists.order, return_residual=wanted,
                                  return_lse=return_lse, check_status=False if check_status == "deferred" else check_status,
                                  **limits)
        if check_status == "deferred":
            ops.post_status(q.device, spacing=ops.STATUS_SPACING)
        if not wanted:
            return res if return_lse else (res, None)
        out, lse, residual = res
        ctx.save_for_backward(q, k, v, out, lse, residual, lists.counts, lists.entries, lists.order, key_lists.counts,
                              key_lists.entries, key_lists.order)
        ctx.limits, ctx.check_status = limits, check_status
        ctx.set_materialize_grads(False)
        if not return_lse:
            return out, None
        ctx.mark_non_differentiable(lse)
        return out, lse

    @staticmethod
    @once_differentiable
    def backward(ctx, dout, _):
        if dout is None:
            return (None,) * 9
        q, k, v, out, lse, residual, *lists = ctx.saved_tensors
        grads = ops.sparse_attn_bwd(dout.contiguous(), q, k, v, out, lse, ops.TileLists(*lists[:3]),
                                    ops.KeyLists(*lists[3:]), residual=residual, check_status=ctx.check_status,
                                    **ctx.limits)
        return tuple(g if need else None for g, need in zip(grads, ctx.needs_input_grad)) + (None,) * 6


def sparse_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, lists: ops.TileLists, key_lists: ops.KeyLists, *,
                     softmax_scale: Optional[float] = None, q_split: Optional[int] = None,
                     kv_len_lo: Optional[int] = None, kv_len_hi: Optional[int] = None,
                     check_status="deferred", return_lse: bool = False):
    """Block-sparse attention of (B, H, N, D) float16 or bfloat16 tensors, differentiable with respect to q, k and v.

    lists, key_lists: `ops.tile_lists` and `ops.key_lists` of the layer's mask; the other arguments are those of
    `ops.sparse_attn_fwd` ("deferred": a call raises for a kernel of an earlier step that gave up a wait, once the copy of its status
    has arrived; copies are queued at most every `ops.STATUS_SPACING` seconds).  return_lse: (out, lse), lse a
    constant.  Tensors that are not contiguous are copied.  What lies between the forward and the backward is q, k, v, the
    output, what rounding took from it, 4 bytes per row and the work lists (of (N / 128)^2 entries of 4 bytes per mask head the
    key lists, half as many the others).

    Where a graph is built, N is at most `_lib.ATTN_BWD_MAX_ROWS`."""
    wanted = _builds_graph(q, k, v)
    if wanted and q.dim() == 4 and q.shape[2] > _lib.ATTN_BWD_MAX_ROWS:
        raise _lib.ModditError(f"gradients of the attention cover {_lib.ATTN_BWD_MAX_ROWS} rows, got {q.shape[2]}: run the "
                               "forward alone under torch.no_grad()")
    limits = dict(softmax_scale=softmax_scale, q_split=q_split, kv_len_lo=kv_len_lo, kv_len_hi=kv_len_hi)
    out, lse = _SparseAttention.apply(q.contiguous(), k.contiguous(), v.contiguous(), lists, key_lists, limits, check_status,
                                      return_lse, wanted)
    return (out, lse) if return_lse else out


class _Prologue(torch.autograd.Function):
    @staticmethod
    def forward(ctx, fused, q_in, k_in, v_in, q_weight, q_bias, k_weight, k_bias, rope_cos, rope_sin, opts):
        if fused is not None:
            q_in, k_in, v_in = fused.split(fused.shape[-1] // 3, dim=-1)
        (q, k, v), _ = ops.qkv_prologue(q_in, k_in, v_in, q_weight=q_weight, q_bias=q_bias, k_weight=k_weight, k_bias=k_bias,
                                        rope_cos=rope_cos, rope_sin=rope_sin, **opts)
        keep = opts["norm"] is not None
        ctx.save_for_backward(fused if keep else None, q_in if keep and fused is None else None,
                              k_in if keep and fused is None else None, q_weight, q_bias, k_weight, k_bias, rope_cos, rope_sin)
        ctx.opts, ctx.fused, ctx.tokens = opts, fused is not None, q_in.shape[1]
        ctx.set_materialize_grads(False)
        return q, k, v

    @staticmethod
    @once_differentiable
    def backward(ctx, *grads):
        fused, q_in, k_in, q_weight, q_bias, k_weight, k_bias, rope_cos, rope_sin = ctx.saved_tensors
        if fused is not None:
            q_in, k_in, _ = fused.split(fused.shape[-1] // 3, dim=-1)
        grads = [None if g is None else g.contiguous() for g in grads]
        given = [g for g in grads if g is not None]
        if not given:
            return (None,) * 11
        needs = ctx.needs_input_grad
        if not ctx.fused:           # an input without a gradient costs nothing, unless its norm's parameters need theirs
            wanted = (needs[1] or needs[4] or needs[5], needs[2] or needs[6] or needs[7], needs[3])
            grads = [g if w else None for g, w in zip(grads, wanted)]
            if all(g is None for g in grads):
                return (None,) * 11
        whole, out = None, None
        if ctx.fused:
            B, H, _, D = given[0].shape
            whole = torch.empty(B, ctx.tokens, 3 * H * D, device=given[0].device, dtype=given[0].dtype)
            out = whole.split(H * D, dim=-1)
            for o, g in zip(out, grads):
                if g is None:
                    o.zero_()
        dx, params = ops.qkv_prologue_bwd(*grads, q_in, k_in, q_weight=q_weight, q_bias=q_bias,
                                          k_weight=k_weight, k_bias=k_bias, rope_cos=rope_cos, rope_sin=rope_sin,
                                          n_tokens=ctx.tokens, out=out, param_grads=any(needs[4:8]), **ctx.opts)
        dx = (None, None, None) if ctx.fused else dx
        return (whole, *dx, params["q_weight"], params["q_bias"], params["k_weight"], params["k_bias"], None, None, None)


def qkv_prologue(q_in: Optional[torch.Tensor] = None, k_in: Optional[torch.Tensor] = None,
                 v_in: Optional[torch.Tensor] = None, *, fused: Optional[torch.Tensor] = None, num_heads: int,
                 norm: Optional[str] = None, q_weight: Optional[torch.Tensor] = None, q_bias: Optional[torch.Tensor] = None,
                 k_weight: Optional[torch.Tensor] = None, k_bias: Optional[torch.Tensor] = None, eps: float = 1e-6,
                 rope_cos: Optional[torch.Tensor] = None, rope_sin: Optional[torch.Tensor] = None,
                 rope_form: str = "elementwise", rope_range: Optional[Tuple[int, int]] = None):
    """(q, k, v) of shape (B, H, S, D) as `ops.qkv_prologue` makes them, differentiable with respect to the projections and the
    norm's parameters (the rotary tables are constants).

    Either q_in, k_in and v_in, (B, S, H*D) each, or `fused`, a contiguous (B, S, 3*H*D) projection whose gradient is written
    in one piece.  The other arguments are those of `ops.qkv_prologue`.  Where a graph is built, norm="rms_all_heads"
    covers up to `_lib.TOKEN_NORM_BWD_MAX_WIDTH` values a token."""
    if (fused is None) == (q_in is None) or (fused is None and (k_in is None or v_in is None)) or \
            (fused is not None and (k_in is not None or v_in is not None)):
        raise ValueError("qkv_prologue: either q_in, k_in and v_in or fused")
    if fused is not None and (fused.dim() != 3 or not fused.is_contiguous() or fused.shape[-1] % (3 * num_heads)):
        raise ValueError(f"fused must be a contiguous (B, S, 3 * {num_heads} * D) tensor")
    width = fused.shape[-1] // 3 if fused is not None else q_in.shape[-1]
    if norm == "rms_all_heads" and width > _lib.TOKEN_NORM_BWD_MAX_WIDTH and \
            _builds_graph(fused, q_in, k_in, v_in, q_weight, q_bias, k_weight, k_bias):
        raise _lib.ModditError(f"gradients of a normalisation over all heads cover {_lib.TOKEN_NORM_BWD_MAX_WIDTH} values a "
                               f"token, got {width}: run the forward alone under torch.no_grad()")
    opts = dict(num_heads=num_heads, norm=None if norm == "none" else norm, eps=eps, rope_form=rope_form, rope_range=rope_range)
    return _Prologue.apply(fused, q_in, k_in, v_in, q_weight, q_bias, k_weight, k_bias, rope_cos, rope_sin, opts)
