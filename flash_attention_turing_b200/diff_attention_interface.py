"""Differential attention: the difference of two softmax maps with a learned weight per head.

The halves of the head dimension of q and k give two maps over the same values::

    A_m = softmax(scale * Q_m K_m^T [+ causal mask]),  m = 1, 2        out = (A_1 - lam_h * A_2) V

Shapes, masks (bottom-right aligned), grouped heads, packed sequences and the KV cache are those of ``flash_attn_func``,
``flash_attn_varlen_func`` and ``flash_attn_with_kvcache``: fp16, head dimension 64 or 128 (maps of 32 or 64).  A model that keeps
2 * nheads query heads of d / 2 and values of d passes ``q.view(b, s, nheads, d)``: the two maps of a head lie next to each other.
``lam`` holds one weight per query head, or a single one for all, fp32 or fp16, and has a gradient.  What a model puts around the
operator (how lam is parametrised, a norm of the heads' outputs) is its own.  ``softmax_scale`` must be at least 1e-6; the weights should
lie well inside fp16's range, the type of the products that they enter.  A row that sees no key is zero; a NaN, or an infinite score, makes NaN of every
row that it reaches.
No counterpart in Cy-47/flash-attention-turing.
"""
from __future__ import annotations

from typing import Optional, Union

import torch

from . import flash_attention_interface as _interface
from .flash_attention_interface import _diff_scale, _gpu, _kvcache_step, _readable


# The classes answer what the native autograd node leaves to them: functorch transforms, tracing, modes, tensor subclasses,
# forward-mode AD, and inputs that are refused.
class FlashDiffAttnFunc(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, lam, softmax_scale, causal, is_grad_enabled):
        scale = _diff_scale(q, softmax_scale)
        q, k, v = (_readable(t) for t in (q, k, v))
        keep = is_grad_enabled and any(t.requires_grad for t in (q, k, v, lam))
        out, lse, *o2 = _gpu().diff_fwd(q, k, v, lam, scale, causal, keep)
        if keep:
            ctx.save_for_backward(q, k, v, lam, out, *o2, lse)
            ctx.softmax_scale, ctx.causal = scale, causal
        return out

    @staticmethod
    def backward(ctx, dout):
        q, k, v, lam, out, o2, lse = ctx.saved_tensors
        dq, dk, dv, dlam = _gpu().diff_bwd(q, k, v, lam, out, o2, lse, _readable(dout), ctx.softmax_scale, ctx.causal)
        return dq, dk, dv, dlam, None, None, None


class FlashDiffAttnVarlenFunc(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, lam, cu_seqlens_q, cu_seqlens_k, max_seqlen_q, max_seqlen_k, softmax_scale, causal,
                is_grad_enabled):
        scale = _diff_scale(q, softmax_scale)
        q, k, v = (_readable(t) for t in (q, k, v))
        keep = is_grad_enabled and any(t.requires_grad for t in (q, k, v, lam))
        out, lse, *o2 = _gpu().diff_varlen_fwd(q, k, v, lam, cu_seqlens_q, cu_seqlens_k, max_seqlen_q, max_seqlen_k, scale, causal, keep)
        if keep:
            ctx.save_for_backward(q, k, v, lam, out, *o2, lse, cu_seqlens_q, cu_seqlens_k)
            ctx.lengths = max_seqlen_q, max_seqlen_k
            ctx.softmax_scale, ctx.causal = scale, causal
        return out

    @staticmethod
    def backward(ctx, dout):
        q, k, v, lam, out, o2, lse, cu_q, cu_k = ctx.saved_tensors
        dq, dk, dv, dlam = _gpu().diff_varlen_bwd(q, k, v, lam, out, o2, lse, _readable(dout), cu_q, cu_k, *ctx.lengths,
                                                  ctx.softmax_scale, ctx.causal)
        return dq, dk, dv, dlam, None, None, None, None, None, None, None


def flash_diff_attn_func(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, lam: torch.Tensor,
                         softmax_scale: Optional[float] = None, causal: bool = False) -> torch.Tensor:
    """q (batch, seqlen_q, nheads, d); k, v (batch, seqlen_k, nheads_k, d); lam (nheads,) or one element -> out like q.
    ``softmax_scale`` defaults to (d / 2) ** -0.5.  Differentiable in q, k, v and lam; every gradient is bitwise reproducible."""
    out = _gpu().diff_attention_dense(q, k, v, lam, softmax_scale, causal)
    return FlashDiffAttnFunc.apply(q, k, v, lam, softmax_scale, causal, torch.is_grad_enabled()) if out is None else out


def flash_diff_attn_varlen_func(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, lam: torch.Tensor, cu_seqlens_q: torch.Tensor,
                                cu_seqlens_k: torch.Tensor, max_seqlen_q: int, max_seqlen_k: int,
                                softmax_scale: Optional[float] = None, causal: bool = False) -> torch.Tensor:
    """Packed sequences: q (total_q, nheads, d); k, v (total_k, nheads_k, d); cu_seqlens_* int32 (batch + 1,) -> out like q.
    Rows outside every sequence are zero in the output and in the gradients and count for nothing, and so are those of a sequence past
    max_seqlen_q."""
    out = _gpu().diff_attention_varlen(q, k, v, lam, cu_seqlens_q, cu_seqlens_k, max_seqlen_q, max_seqlen_k, softmax_scale, causal)
    if out is not None:
        return out
    return FlashDiffAttnVarlenFunc.apply(q, k, v, lam, cu_seqlens_q, cu_seqlens_k, max_seqlen_q, max_seqlen_k, softmax_scale,
                                         causal, torch.is_grad_enabled())


def flash_diff_attn_with_kvcache(
    q: torch.Tensor,
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    lam: torch.Tensor,
    k: Optional[torch.Tensor] = None,
    v: Optional[torch.Tensor] = None,
    cache_seqlens: Optional[Union[torch.Tensor, int]] = None,
    cache_batch_idx: Optional[torch.Tensor] = None,
    block_table: Optional[torch.Tensor] = None,
    softmax_scale: Optional[float] = None,
    causal: bool = False,
    num_splits: int = 0,
) -> torch.Tensor:
    """Inference step against a KV cache: appends ``k``/``v`` in place at ``cache_seqlens`` and attends ``q`` against the first
    ``cache_seqlens + seqlen_new`` tokens.  The caches (contiguous or paged), the arguments and their checks are those of
    ``flash_attn_with_kvcache``, and a cache may be used by both; ``num_splits`` is honoured as there for up to 64 queries times heads of a KV
    head and is an upper bound for more.  Not differentiable."""
    if not isinstance(lam, torch.Tensor):
        raise TypeError("lam must be a torch.Tensor")
    # An ordinary decode step: the binding makes the same checks, and returns None for whatever it does not take as it is or would
    # refuse, before anything has been done.  (1 x 1500 tokens: 17.4 -> 14.9 us a call, whose host waits for the device's answer.)
    if _interface.HOST_CAPACITY_CHECK and cache_batch_idx is None and isinstance(cache_seqlens, torch.Tensor) and q.is_cuda and q.shape[-1] in (64, 128):
        r = _gpu().diff_kvcache_checked(q, k_cache, v_cache, lam, k, v, cache_seqlens, None, block_table,
                                        _diff_scale(q, softmax_scale), causal, num_splits)
        if r is not None and r[2]:
            return r[0]
    return _kvcache_step(q, k_cache, v_cache, k, v, cache_seqlens, cache_batch_idx, block_table, softmax_scale, causal, num_splits,
                         False, lam=lam)
