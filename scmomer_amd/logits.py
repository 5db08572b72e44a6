"""What a program reads off a model's logits, and what it trains them towards, for any number of classes: log
probabilities of given tokens with entropy and top alternatives (token_logprobs).  The RNA model's own masked cross
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


def _shaped(shape, outs):
    lp, ent, lse, tlp, tix = outs
    return (lp if lp is None else lp.view(shape), ent if ent is None else ent.view(shape), lse.view(shape),
            tlp if tlp is None else tlp.view(*shape, tlp.shape[1]), tix if tix is None else tix.view(*shape, tix.shape[1]))


class _TokenLogprobsFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, targets, k, temperature, ignore_index, entropy):
        *outs, tape = ops.score_fwd(logits, targets, k, temperature, ignore_index, entropy, tape=True)
        ctx.set_materialize_grads(False)
        ctx.opts = (temperature, ignore_index)
        ctx.save_for_backward(logits, targets, tape, outs[1], outs[4])
        if k:
            ctx.mark_non_differentiable(outs[4])
        return _shaped(logits.shape[:-1], outs)

    @staticmethod
    @once_differentiable
    def backward(ctx, g_logprob, g_entropy, g_lse, g_top, _):
        logits, targets, tape, entropy, top_index = ctx.saved_tensors
        dx = ops.score_bwd(logits, targets, tape, entropy, top_index, g_logprob, g_entropy, g_lse, g_top, *ctx.opts)
        return dx.view(logits.shape), None, None, None, None, None


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
    return TokenLogprobs(*_shaped(logits.shape[:-1], ops.score_fwd(logits, targets, k, temperature, ignore_index, entropy)[:5]))
