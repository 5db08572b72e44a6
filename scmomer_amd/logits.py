"""What a program reads off a model's logits, and what it trains them towards, for any number of classes: log
probabilities of given tokens with entropy and top alternatives (token_logprobs), and distillation from a teacher's top
log probabilities (topk_distillation, topk_distillation_grad).  The RNA model's own masked cross
entropy over its at most eight expression classes is s1.masked_cross_entropy.

Differentiable means once and in reverse mode: under forward-mode differentiation, a tracer (torch.jit.trace, make_fx),
torch.func's transforms or with tensor subclasses that have a dispatch of their own they raise NotImplementedError, and so
does their backward pass.

A backward pass of these under capture into a graph is refused while an eager graph on the default stream holds a leaf that
it reaches (that leaf's gradient would have to join that stream).
"""
from __future__ import annotations

from typing import NamedTuple, Optional

import torch

from . import _lib


class TokenLogprobs(NamedTuple):
    """Per row of the logits; ``logprob`` is None without targets, ``entropy`` where it is not asked for, the
    alternatives for k = 0."""
    logprob: Optional[torch.Tensor]       # f32 [...]
    entropy: Optional[torch.Tensor]       # f32 [...]
    lse: torch.Tensor                     # f32 [...]: log of the sum of exponentials
    top_logprob: Optional[torch.Tensor]   # f32 [..., k], descending
    top_index: Optional[torch.Tensor]     # int64 [..., k]


def token_logprobs(logits: torch.Tensor, targets: Optional[torch.Tensor] = None, *, k: int = 0, temperature: float = 1.0,
                   ignore_index: int = -100, entropy: bool = True) -> TokenLogprobs:
    """Log probabilities under softmax(logits / temperature), over the last dimension of logits [..., V].

    logits: f32, bf16 or fp16 on the GPU, any row stride; targets: int64 [...] or None; temperature: finite and at least
    2^-126 (below, its reciprocal leaves the range of f32).  Everything is computed in f32 and returned in f32.
    ``logprob``: of the target token, 0 where the target is ``ignore_index``, NaN where it is any other number outside
    [0, V).  ``top_index`` / ``top_logprob``: the k <= min(64, V) most likely tokens in descending order, equal logits by
    ascending index (NaN counts as largest).  A row that is -inf throughout has lse and log probabilities -inf, entropy 0
    and no gradient; a row with NaN or +inf is NaN.

    Differentiable once in the logits, through every output but ``top_index`` (the choice of the alternatives is a
    constant, as for torch.topk).  Two calls with the same logits give the same bits; the same row in a call of another
    number of rows may differ in the last ones (how its sum is split over threads depends on that number)."""
    return TokenLogprobs(*_lib.torch_ops.token_logprobs(logits, targets, k, temperature, ignore_index, entropy))


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
    temperature: as for token_logprobs.

    Differentiable once, in the logits only.  The result does not depend on the order in which workgroups run; a row's last
    bits may depend on the number of rows in the call, as for token_logprobs."""
    return _lib.torch_ops.topk_distillation(logits, top_index, top_logprob, temperature, tail, weight, reduction)


def topk_distillation_grad(logits: torch.Tensor, top_index: torch.Tensor, top_logprob: torch.Tensor, *,
                           temperature: float = 1.0, tail: bool = True, weight: Optional[torch.Tensor] = None,
                           reduction: str = "mean", scale: float = 1.0):
    """(loss, scale * d loss / d logits) of topk_distillation ('mean' or 'sum') in one pass over the logits, for a loop
    that runs the model's backward itself: ``loss, d = topk_distillation_grad(logits, ..., scale=1 / grad_acc)``,
    ``logits.backward(d)``.  The gradient has the logits' type and shape."""
    return _lib.torch_ops.topk_distillation_grad(logits, top_index, top_logprob, temperature, tail, weight, reduction, scale)
