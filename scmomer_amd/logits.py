"""What a program reads off a model's logits, and what it trains them towards, for any number of classes: log
probabilities of given tokens with entropy and top alternatives (token_logprobs), and distillation from a teacher's top
log probabilities (topk_distillation, topk_distillation_grad).  The RNA model's own masked cross
entropy over its at most eight expression classes is s1.masked_cross_entropy.
"""
from __future__ import annotations

from typing import NamedTuple, Optional

import torch
from torch.autograd.function import once_differentiable

from . import ops


class TokenLogprobs(NamedTuple):
    """Per row of the logits; ``logprob`` is None without targets, ``entropy`` where it is not asked for, the
    alternatives for k = 0."""
    logprob: Optional[torch.Tensor]       # f32 [...]
    entropy: Optional[torch.Tensor]       # f32 [...]
    lse: torch.Tensor                     # f32 [...]: log of the sum of exponentials
    top_logprob: Optional[torch.Tensor]   # f32 [..., k], descending
    top_index: Optional[torch.Tensor]     # int64 [..., k]


def _shaped(logits, lp, ent, lse, tlp, tix):
    if logits.dim() == 2:
        return lp, ent, lse, tlp, tix
    shape = logits.shape[:-1]
    return (lp if lp is None else lp.view(shape), ent if ent is None else ent.view(shape), lse.view(shape),
            tlp if tlp is None else tlp.view(*shape, tlp.shape[1]), tix if tix is None else tix.view(*shape, tix.shape[1]))


class _TokenLogprobsFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, targets, k, temperature, ignore_index, entropy):
        lp, ent, lse, tlp, tix, tape = ops.score_fwd(logits, targets, k, temperature, ignore_index, entropy, tape=True)
        ctx.set_materialize_grads(False)
        ctx.opts = (temperature, ignore_index)
        ctx.save_for_backward(logits, targets, ent, tix, tape)
        if k:
            ctx.mark_non_differentiable(tix)
        return _shaped(logits, lp, ent, lse, tlp, tix)

    @staticmethod
    def backward(ctx, g_logprob, g_entropy, g_lse, g_top, _):
        if torch.is_grad_enabled():
            return _TokenLogprobsFn._once(ctx, g_logprob, g_entropy, g_lse, g_top, _)
        logits, targets, entropy, top_index, tape = ctx.saved_tensors
        dx = ops.score_bwd(logits, targets, tape, entropy, top_index, g_logprob, g_entropy, g_lse, g_top, *ctx.opts)
        return dx if logits.dim() == 2 else dx.view(logits.shape), None, None, None, None, None

    @staticmethod
    @once_differentiable
    def _once(ctx, *grads):      # under create_graph: what comes back refuses to be differentiated again
        return _TokenLogprobsFn.backward(ctx, *grads)


def token_logprobs(logits: torch.Tensor, targets: Optional[torch.Tensor] = None, *, k: int = 0, temperature: float = 1.0,
                   ignore_index: int = -100, entropy: bool = True) -> TokenLogprobs:
    """Log probabilities under softmax(logits / temperature), over the last dimension of logits [..., V].

    logits: f32, bf16 or fp16 on the GPU, any row stride; targets: int64 [...] or None.  Everything is computed in f32
    and returned in f32.  ``logprob``: of the target token, 0 where the target is ``ignore_index``, NaN where it is any
    other number outside [0, V).  ``top_index`` / ``top_logprob``: the k <= min(64, V) most likely tokens in descending
    order, equal logits by ascending index (NaN counts as largest).  A row that is -inf throughout has lse and log
    probabilities -inf, entropy 0 and no gradient; a row with NaN or +inf is NaN.

    Differentiable once in the logits, through every output but ``top_index`` (the choice of the alternatives is a
    constant, as for torch.topk)."""
    if torch.is_grad_enabled() and logits.requires_grad:
        return TokenLogprobs(*_TokenLogprobsFn.apply(logits, targets, k, temperature, ignore_index, entropy))
    return TokenLogprobs(*_shaped(logits, *ops.score_fwd(logits, targets, k, temperature, ignore_index, entropy)[:5]))


class _TopkDistillFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, top_index, top_logprob, temperature, tail, weight, reduction):
        op = ops.TopkDistill(logits, top_index, top_logprob, temperature, tail, weight, reduction)
        rows, loss, wsum, tape = op.forward(reduction != "none", True)
        ctx.opts = (temperature, tail, reduction)
        ctx.save_for_backward(logits, top_index, top_logprob, weight, wsum, tape)
        return loss if loss is not None else rows if logits.dim() == 2 else rows.view(logits.shape[:-1])

    @staticmethod
    def backward(ctx, gloss):
        if torch.is_grad_enabled():
            return _TopkDistillFn._once(ctx, gloss)
        logits, top_index, top_logprob, weight, wsum, tape = ctx.saved_tensors
        temperature, tail, reduction = ctx.opts
        dx = ops.TopkDistill.again(logits, top_index, top_logprob, temperature, tail, weight, reduction).backward(gloss, wsum, tape)
        return dx if logits.dim() == 2 else dx.view(logits.shape), None, None, None, None, None, None

    @staticmethod
    @once_differentiable
    def _once(ctx, gloss):      # under create_graph: what comes back refuses to be differentiated again
        return _TopkDistillFn.backward(ctx, gloss)


def topk_distillation(logits: torch.Tensor, top_index: torch.Tensor, top_logprob: torch.Tensor, *, temperature: float = 1.0,
                      tail: bool = True, weight: Optional[torch.Tensor] = None, reduction: str = "mean") -> torch.Tensor:
    """KL divergence from a teacher's top log probabilities to softmax(logits / temperature).

    logits [..., V]: f32, bf16 or fp16 on the GPU, any row stride; top_index int64 [..., k], top_logprob f32 [..., k],
    1 <= k <= 64: the teacher's entries at the same temperature, as token_logprobs returns them (a negative index is an
    entry not used; one named twice counts with both probabilities; one outside the vocabulary makes the row NaN).
    ``tail``: what the entries leave of the teacher's mass is one more class against the student's mass on all other
    tokens; otherwise the entries are renormalised.  ``weight`` f32 [...]: rows of weight 0 (padding) are not looked at.
    reduction 'mean' divides by the sum of the weights (nan when that is 0), 'none' returns weight * loss per row.  The
    loss is f32 and not multiplied by temperature^2.  A row of -inf throughout counts with loss and gradient 0.

    Differentiable once, in the logits only.  The result does not depend on the order in which workgroups run."""
    if torch.is_grad_enabled() and logits.requires_grad:
        return _TopkDistillFn.apply(logits, top_index, top_logprob, temperature, tail, weight, reduction)
    op = ops.TopkDistill(logits, top_index, top_logprob, temperature, tail, weight, reduction)
    rows, loss, _, _ = op.forward(reduction != "none", False)
    return loss if loss is not None else rows.view(logits.shape[:-1])


def topk_distillation_grad(logits: torch.Tensor, top_index: torch.Tensor, top_logprob: torch.Tensor, *,
                           temperature: float = 1.0, tail: bool = True, weight: Optional[torch.Tensor] = None,
                           reduction: str = "mean", scale: float = 1.0):
    """(loss, scale * d loss / d logits) of topk_distillation ('mean' or 'sum') in one pass over the logits, for a loop
    that runs the model's backward itself: ``loss, d = topk_distillation_grad(logits, ..., scale=1 / grad_acc)``,
    ``logits.backward(d)``.  The gradient has the logits' type and shape."""
    if reduction == "none":
        raise ValueError("topk_distillation_grad: reduction must be 'mean' or 'sum'")
    loss, dx = ops.TopkDistill(logits.detach(), top_index, top_logprob, temperature, tail, weight, reduction).step(scale)
    return loss, dx if logits.dim() == 2 else dx.view(logits.shape)
