"""Differentiable forms of the attention calls and of what comes right before them in a layer.

  flash_attention         ops.flash_fwd with ops.flash_bwd
  block_sparse_attention  ops.block_sparse_fwd with ops.block_sparse_bwd
  qk_norm_rope            ops.qk_norm_rope with ops.qk_norm_rope_bwd

For training or distilling a layer under its predicted masks. The step machine
(`SparseAttentionWithMap`) and `AttentionSparseEngine` serve inference and return outputs that
carry no gradient. First derivatives only.

A backward pass that is captured into a HIP graph needs leaves of its own: torch ties a leaf's
gradient accumulation to the stream of the first graph that reached it, so an eager graph of the
same leaves that still lives breaks the capture. `torch.autograd.grad` on detached leaves, or the
functions of `ops` without autograd, capture as they are.
"""
from __future__ import annotations

import torch
from torch.autograd.function import once_differentiable

from . import ops


class _Attention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, tiles, key_tiles, scale):
        if tiles is None:
            out, lse = ops.flash_fwd(q, k, v, scale, return_lse=True)
        else:
            out, lse = ops.block_sparse_fwd(q, k, v, tiles, scale, return_lse=True)
        ctx.save_for_backward(q, k, v, out, lse)
        ctx.tiles, ctx.key_tiles, ctx.scale = tiles, key_tiles, scale
        ctx.set_materialize_grads(False)
        return out, lse

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_out, grad_lse):
        q, k, v, out, lse = ctx.saved_tensors
        if grad_out is None and grad_lse is None:
            return (None,) * 6
        if grad_out is None:
            grad_out = torch.zeros_like(out)
        if ctx.tiles is None:
            grads = ops.flash_bwd(q, k, v, out, lse, grad_out, ctx.scale, grad_lse)
        else:
            grads = ops.block_sparse_bwd(q, k, v, out, lse, grad_out, ctx.tiles, ctx.scale, grad_lse,
                                         ctx.key_tiles)
        return (*(g if need else None for g, need in zip(grads, ctx.needs_input_grad)), None, None, None)


def flash_attention(query, key, value, softmax_scale=None, return_lse=False):
    """Differentiable dense attention over all keys, (B,H,S,D) bf16/fp16; O, or (O, LSE) with
    `return_lse`. The LSE (B,H,S) fp32 is differentiable too."""
    out, lse = _Attention.apply(query, key, value, None, None, softmax_scale)
    return (out, lse) if return_lse else out


def block_sparse_attention(query, key, value, tiles: ops.TileList, softmax_scale=None, return_lse=False,
                           key_tiles: ops.KeyTileList | None = None):
    """Differentiable attention restricted to the active key tiles of `tiles`
    (`ops.mask_to_tiles`). `key_tiles` (`ops.transpose_tiles`): kept by a caller that trains under
    one mask for several steps, else the backward pass builds it. The lists must keep their values
    until the backward pass has run."""
    out, lse = _Attention.apply(query, key, value, tiles, key_tiles, softmax_scale)
    return (out, lse) if return_lse else out


class _QkNormRope(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, q_weight, k_weight, q_bias, k_bias, cos, sin, opts):
        out = ops.qk_norm_rope(q, k, q_weight=q_weight, k_weight=k_weight, q_bias=q_bias, k_bias=k_bias,
                               cos=cos, sin=sin, **opts)
        ctx.save_for_backward(q, k, q_weight, k_weight, q_bias, k_bias, cos, sin)
        ctx.opts = opts
        ctx.set_materialize_grads(False)
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_q, grad_k):
        q, k, q_weight, k_weight, q_bias, k_bias, cos, sin = ctx.saved_tensors
        if grad_q is None and grad_k is None:
            return (None,) * 9
        grad_q = torch.zeros_like(q) if grad_q is None else grad_q
        grad_k = torch.zeros_like(k) if grad_k is None else grad_k
        dq, dk, *sums = ops.qk_norm_rope_bwd(q, k, grad_q, grad_k, q_weight=q_weight, k_weight=k_weight,
                                             q_bias=q_bias, k_bias=k_bias, cos=cos, sin=sin, **ctx.opts)
        sums = (None if t is None else t.to(like.dtype)
                for t, like in zip(sums, (q_weight, k_weight, q_bias, k_bias)))
        grads = (dq, dk, *sums)
        return (*(g if need else None for g, need in zip(grads, ctx.needs_input_grad)), None, None, None)


def qk_norm_rope(query, key, *, norm="rms", across_heads=False, eps=1e-6, q_weight=None, k_weight=None,
                 q_bias=None, k_bias=None, cos=None, sin=None, rope_offset=0, interleaved=True):
    """Differentiable `ops.qk_norm_rope`: norm of queries and keys and the rotation of their
    positions in one pass; returns (query', key'). The tables carry no gradient."""
    if any(t is not None and t.requires_grad for t in (cos, sin)):
        raise ValueError("qk_norm_rope: cos and sin carry no gradient; detach them")
    return _QkNormRope.apply(query, key, q_weight, k_weight, q_bias, k_bias, cos, sin,
                             dict(norm=norm, across_heads=across_heads, eps=eps, rope_offset=rope_offset,
                                  interleaved=interleaved))
