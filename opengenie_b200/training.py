"""Differentiable attention and Q/K norm + rotation for adapting the video block: the training pass of
``ltx_ops.attention_with_lse`` / ``attention_backward`` and ``fused_qk_norm_rope`` / ``fused_qk_norm_rope_backward`` as
torch autograd functions.

Everything else of a training step (projections, losses, the optimizer) is the caller's torch code.  The attention
backend (``attention_backend.B200NativeAttention``) comes here by itself when an input requires a gradient.

In a CUDA graph: capture the explicit functions of ``ltx_ops`` (forward, backward), which know nothing of autograd.  A
captured ``backward()`` is bound to torch's own rule that no graph of an earlier eager pass over the same leaves may be
alive then, since their gradient accumulators belong to that pass's stream.
"""

from __future__ import annotations

import torch
from torch.autograd.function import once_differentiable

from . import ltx_ops


def _addressable(grad: torch.Tensor) -> torch.Tensor:
    """A gradient as the kernels read it: torch hands over expanded or transposed ones (``out.sum().backward()``)."""
    return grad if ltx_ops._rows(grad) is not None else grad.clone(memory_format=torch.contiguous_format)


class _Attention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, q_lengths, kv_lengths, heads, options):
        out, lse = ltx_ops.attention_with_lse(q, k, v, heads, q_lengths=q_lengths, kv_lengths=kv_lengths, **options)
        ctx.save_for_backward(q, k, v, out, lse, q_lengths, kv_lengths)
        ctx.heads, ctx.options = heads, options
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, dout):
        q, k, v, out, lse, q_lengths, kv_lengths = ctx.saved_tensors
        grads = ltx_ops.attention_backward(_addressable(dout), q, k, v, out, lse, ctx.heads, q_lengths=q_lengths,
                                           kv_lengths=kv_lengths, **ctx.options)
        return *grads, None, None, None, None


def attention(
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    heads: int,
    *,
    kv_heads: int | None = None,
    softmax_scale: float | None = None,
    causal_block: int = 0,
    q_lengths: torch.Tensor | None = None,
    kv_lengths: torch.Tensor | None = None,
) -> torch.Tensor:
    """``ltx_ops.attention_with_lse`` (its arguments and masks) as a differentiable function of q, k and v."""
    options = dict(kv_heads=kv_heads, softmax_scale=softmax_scale, causal_block=causal_block)
    return _Attention.apply(q, k, v, q_lengths, kv_lengths, heads, options)


class _QKNormRope(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, q_weight, k_weight, cos, sin, eps, heads, options):
        ctx.save_for_backward(q, k, q_weight, k_weight, cos, sin)
        ctx.eps, ctx.heads, ctx.options = eps, heads, options
        return ltx_ops.fused_qk_norm_rope(q, k, q_weight, k_weight, eps, cos, sin, heads, **options)

    @staticmethod
    @once_differentiable
    def backward(ctx, dq_out, dk_out):
        q, k, q_weight, k_weight, cos, sin = ctx.saved_tensors
        dq, dk, dqw, dkw = ltx_ops.fused_qk_norm_rope_backward(
            _addressable(dq_out), _addressable(dk_out), q, k, q_weight, k_weight, ctx.eps, cos, sin, ctx.heads,
            **ctx.options)
        if dqw is not None:  # torch wants a weight's gradient in the weight's type
            dqw, dkw = dqw.to(q_weight.dtype), dkw.to(k_weight.dtype)
        return dq, dk, dqw, dkw, None, None, None, None, None


def qk_norm_rope(
    q: torch.Tensor,
    k: torch.Tensor,
    q_weight: torch.Tensor | None,
    k_weight: torch.Tensor | None,
    eps: float,
    cos: torch.Tensor,
    sin: torch.Tensor,
    heads: int,
    *,
    kv_heads: int | None = None,
    norm: str = "head",
    interleaved: bool = False,
) -> tuple[torch.Tensor, torch.Tensor]:
    """``ltx_ops.fused_qk_norm_rope`` (its arguments and layouts) as a differentiable function of q, k and the weights;
    the angle tables are constants.  The weights' gradients are summed in 32 bits and rounded once to their type."""
    options = dict(kv_heads=kv_heads, norm=norm, interleaved=interleaved)
    return _QKNormRope.apply(q, k, q_weight, k_weight, cos, sin, eps, heads, options)


__all__ = ["attention", "qk_norm_rope"]
