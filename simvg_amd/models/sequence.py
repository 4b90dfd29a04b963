"""Differentiable forms of the sequence operators (`hip_ops.qk_norm_rope_*`, `packed_attn_*`, `vocab_ce_*`): what a decoder over this
path's image and text tokens is trained with.  PyTorch autograd is the tape only, as in `heads/functions.py`.

    plan = packed_plan(cu_seqlens, T)                                   # once for a batch, for all layers
    q, k = qk_norm_rope(q, k, pos, inv_freq, sections, gq, gk)          # [T, H, D]
    o = packed_attention(q, k, v, plan)                                 # causal, grouped heads
    loss = vocab_cross_entropy(x, w, target, bias)                      # the logits are never stored

All run on the current stream and may be captured into a HIP graph, forward and backward (a captured backward pass must not find an
eager graph of the same leaves alive: torch ends the process then).  A second derivative is refused.
"""
import torch
from torch.autograd.function import once_differentiable

from .. import hip_ops as ops
from ..hip_ops import PackedPlan, packed_plan          # noqa: F401  (part of this module's interface)

__all__ = ["PackedPlan", "packed_plan", "qk_norm_rope", "packed_attention", "vocab_cross_entropy"]


def _rows(t):
    """a gradient with rows of 16-byte chunks (autograd may hand over an expanded or transposed one, or a part of a larger one)"""
    fits = t.stride(-1) == 1 and all(s % 8 == 0 for s in t.stride()[:-1]) and t.data_ptr() % 16 == 0
    return t if fits else t.clone(memory_format=torch.contiguous_format)


class QKNormRope(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, pos, inv_freq, sections, gq, gk, eps, interleaved):
        ctx.save_for_backward(q, k, pos, inv_freq, gq, gk)
        ctx.args = (sections, eps, interleaved)
        return ops.qk_norm_rope_fwd(q, k, pos, inv_freq, sections, gq, gk, eps, interleaved)

    @staticmethod
    @once_differentiable
    def backward(ctx, dq, dk):
        q, k, pos, inv_freq, gq, gk = ctx.saved_tensors
        sections, eps, interleaved = ctx.args
        dq, dk, dgq, dgk = ops.qk_norm_rope_bwd(_rows(dq), _rows(dk), q, k, pos, inv_freq, sections, gq, gk, eps, interleaved)
        return dq, dk, None, None, None, dgq, dgk, None, None


class PackedAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, plan, causal, scale):
        out, lse = ops.packed_attn_fwd(q, k, v, plan, causal, scale)
        ctx.save_for_backward(q, k, v, out, lse)
        ctx.args = (plan, causal, scale)
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, dout):
        q, k, v, out, lse = ctx.saved_tensors
        plan, causal, scale = ctx.args
        return (*ops.packed_attn_bwd(q, k, v, out, lse, _rows(dout), plan, causal, scale), None, None, None)


class VocabCrossEntropy(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w, target, bias, ignore_index):
        loss, lse = ops.vocab_ce_fwd(x, w, target, bias, ignore_index)
        ctx.save_for_backward(x, w, target, bias, lse)
        ctx.ignore_index = ignore_index
        return loss

    @staticmethod
    @once_differentiable
    def backward(ctx, dloss):
        x, w, target, bias, lse = ctx.saved_tensors
        dx, dw, dbias = ops.vocab_ce_bwd(x, w, target, lse, dloss.contiguous(), bias, ctx.ignore_index)
        return dx, dw, None, dbias, None


class ReducedLoss(torch.autograd.Function):
    @staticmethod
    def forward(ctx, loss, target, ignore_index, mean):
        total, count = ops.vocab_ce_reduce(loss, target, ignore_index, mean)
        ctx.save_for_backward(count)
        ctx.rows = loss.shape
        return total

    @staticmethod
    @once_differentiable
    def backward(ctx, dtotal):
        return (dtotal / ctx.saved_tensors[0]).expand(ctx.rows), None, None, None


def qk_norm_rope(q, k, pos, inv_freq, sections, gq=None, gk=None, eps=1e-6, interleaved=False):
    """`hip_ops.qk_norm_rope_fwd` with gradients for q, k and the norm weights"""
    return QKNormRope.apply(q, k, pos, inv_freq, tuple(sections), gq, gk, eps, interleaved)


def packed_attention(q, k, v, plan, causal=True, scale=None):
    """`hip_ops.packed_attn_fwd` with gradients for q, k and v; rows behind the last sequence are zeros, and so are their gradients"""
    return PackedAttention.apply(q, k, v, plan, causal, scale)


def vocab_cross_entropy(x, w, target, bias=None, ignore_index=-100, reduction="mean"):
    """`hip_ops.vocab_ce_fwd` with gradients for x, w and the bias.  reduction: "mean" over the rows that are not ignored (NaN without any),
    "sum" or "none"."""
    if reduction not in ("mean", "sum", "none"):
        raise ValueError(f"reduction must be mean, sum or none, got {reduction!r}")
    loss = VocabCrossEntropy.apply(x, w, target, bias, ignore_index)
    return loss if reduction == "none" else ReducedLoss.apply(loss, target, ignore_index, reduction == "mean")
