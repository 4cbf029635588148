"""Function layer: ``sdpAttention`` with the reference's signature and a working
backward.

Mirrors function::sdpAttention / FuncSDPAttention
(src/Function/FuncNNLayer.h:229-268, 298-302): same argument order and meaning
(query, key, value, isCausal, attnMask, dropoutP, scale), same default scale
1/sqrt(D), same top-left causal alignment, same assertion that isCausal and a
mask are mutually exclusive, same mask semantics (Bool: true = the key takes
part; otherwise added to the scaled scores; broadcast against [B, H, L, S],
src/Function/FuncNNLayer.h:249-256).  Differences, all forced by the fused path:
  * forward saves (O, LSE) for backward, as the reference's implemented
    backwards save what they need (AutogradContext::pushData,
    src/Tensor/Function.h:24-31);
  * backward exists (the reference traps, FuncNNLayer.h:267) and hands dQ, dK, dV
    to autograd, which accumulates them like AutogradMeta::addGrad
    (src/Tensor/AutogradMeta.cpp:29-43);
  * ``kvLens`` (int32 [B]) is the cheap form of the reference's per-batch length
    mask and may be combined with isCausal; isCausal may also be the string
    "bottom-right" (a chunk of new queries at the end of the keys);
  * a query row with no participating key gives O = 0 (the reference gives NaN);
  * the mask receives no gradient; dropoutP must be 0 (dropout stays on the
    reference's generic-op composition, which this package does not contain).
"""
import torch

from . import _capi, op


class FuncSDPAttention(torch.autograd.Function):
    """The differentiable operator as a Python autograd function: what a trace records, and what torch refuses under
    forward-mode differentiation and functorch's transforms.  Ordinary calls take the native node with the same kernels
    (AttentionBackward in csrc/binding.cpp), which costs less host time."""

    @staticmethod
    def forward(ctx, query, key, value, isCausal, kvLens, scale, attnMask=None):
        needs_grad = any(ctx.needs_input_grad[:3])
        o, lse = op.sdpAttentionFwd(query, key, value, isCausal, scale, kvLens, needLse=needs_grad, attnMask=attnMask)
        if needs_grad:
            ctx.save_for_backward(query, key, value, o, lse)
            ctx.isCausal, ctx.scale, ctx.kvLens, ctx.attnMask = isCausal, scale, kvLens, attnMask
        return o

    @staticmethod
    def backward(ctx, grad):
        query, key, value, o, lse = ctx.saved_tensors
        if grad.stride(3) != 1 or grad.size(2) > 1 and grad.stride(2) == 0:  # (one value, or one row, expanded)
            grad = grad.contiguous()
        dq, dk, dv = op.sdpAttentionBwd(grad, query, key, value, o, lse, ctx.isCausal, ctx.scale, ctx.kvLens,
                                        needs=ctx.needs_input_grad[:3], attnMask=ctx.attnMask)
        return dq, dk, dv, None, None, None, None


class FuncSDPAttentionPacked(torch.autograd.Function):
    """As FuncSDPAttention, for packed sequences (the native node is PackedBackward)."""

    @staticmethod
    def forward(ctx, query, key, value, cuSeqlens, cuSeqlensK, isCausal, scale, status=None):
        needs_grad = any(ctx.needs_input_grad[:3])
        o, lse = op.sdpAttentionPackedFwd(query, key, value, cuSeqlens, isCausal, scale, cuSeqlensK, needLse=needs_grad, status=status)
        if needs_grad:
            ctx.save_for_backward(query, key, value, o, lse, cuSeqlens, cuSeqlensK)
            ctx.isCausal, ctx.scale, ctx.status = isCausal, scale, status
        return o

    @staticmethod
    def backward(ctx, grad):
        query, key, value, o, lse, cuSeqlens, cuSeqlensK = ctx.saved_tensors
        dq, dk, dv = op.sdpAttentionPackedBwd(grad, query, key, value, o, lse, cuSeqlens, ctx.isCausal, ctx.scale, cuSeqlensK,
                                              needs=ctx.needs_input_grad[:3], status=ctx.status)
        return dq, dk, dv, None, None, None, None, None


def sdpAttentionPacked(query, key, value, cuSeqlens, isCausal=False, scale=None, cuSeqlensK=None, status=None):
    """Attention over sequences packed behind one another without padding, differentiable: query [rows, Hq, D], key and
    value [rows, Hkv, D], float16 / bfloat16; sequence n is the rows cuSeqlens[n] to cuSeqlens[n + 1] (int32 [N + 1] on the device).

    With cuSeqlensK keys have lengths of their own, and isCausal="bottom-right" aligns each sequence's queries to the end of its
    keys.  Sequences may be empty; rows of no sequence (behind the last, say) give O = 0 and zero gradients.  The reference has padded
    batches only; each sequence here is what sdpAttention makes of it alone.

    Offsets that fall, are negative or lie beyond the rows give zeros and zero gradients, and set bit 16 of status (int32 [1]), if there
    is one, in both passes; its bit 1 stands for a device-side wait that expired."""
    if not isinstance(isCausal, str):
        isCausal = bool(isCausal)
    o = _capi.native().sdp_attention_packed(query, key, value, cuSeqlens, cuSeqlensK, op._causal_mode(isCausal), scale, status)
    if o is NotImplemented:
        scale = op.default_scale(query.shape[-1]) if scale is None else float(scale)
        o = FuncSDPAttentionPacked.apply(query, key, value, cuSeqlens, cuSeqlensK, isCausal, scale, status)
    return o


def sdpAttention(query, key, value, isCausal=False, attnMask=None, dropoutP=0.0, scale=None, kvLens=None):
    """Drop-in for function::sdpAttention (src/Function/FuncNNLayer.h:298-302)."""
    if isCausal and attnMask is not None:
        raise AssertionError("isCausal and attnMask are mutually exclusive (FuncNNLayer.h:242)")
    if dropoutP > 0.0:
        raise NotImplementedError("dropoutP > 0 is not on the fused path")
    if not isinstance(isCausal, str):
        isCausal = bool(isCausal)
    o = _capi.native().sdp_attention(query, key, value, op._causal_mode(isCausal), kvLens, scale, attnMask)
    if o is NotImplemented:
        scale = op.default_scale(query.shape[-1]) if scale is None else float(scale)
        o = FuncSDPAttention.apply(query, key, value, isCausal, kvLens, scale, None if attnMask is None else attnMask.detach())
    return o
