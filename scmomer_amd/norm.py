"""LayerNorm over rows of any width up to 16384 in f32, bf16 or fp16, as a differentiable function: the norms outside
the Performer stack (a student's hidden layers, the norm before a head), where the stack's own kernels
(ops.ln_fwd / ln_bwd: f32 residual stream, at most 256 columns) do not apply.
"""
from __future__ import annotations

from typing import Optional

import torch
from torch.autograd.function import once_differentiable

from . import ops


class _LayerNormFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps, out_dtype):
        y, stats = ops.norm_fwd(x, weight, bias, eps, out_dtype)
        ctx.save_for_backward(x, weight, stats)
        return y if x.dim() == 2 else y.view(x.shape)

    @staticmethod
    def backward(ctx, dy):
        if torch.is_grad_enabled():
            return _LayerNormFn._once(ctx, dy)
        x, weight, stats = ctx.saved_tensors
        want = ctx.needs_input_grad
        dx, dw, db = ops.norm_bwd(dy, x, stats, weight, want[0], want[1], want[2])
        return dx if dx is None or x.dim() == 2 else dx.view(x.shape), dw, db, None, None

    @staticmethod
    @once_differentiable
    def _once(ctx, dy):      # under create_graph: what comes back refuses to be differentiated again
        return _LayerNormFn.backward(ctx, dy)


def layer_norm(x: torch.Tensor, weight: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None,
               eps: float = 1e-5, *, out_dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """(x - mean) / sqrt(var + eps) * weight + bias over the last dimension D of x [..., D].

    x: f32, bf16 or fp16 on the GPU, 1 <= D <= 16384, any row stride (other layouts are copied first); weight, bias:
    f32 [D] or None (1, 0).  The result has x's type, or bfloat16 from f32 with ``out_dtype=torch.bfloat16``;
    statistics and the gradients of weight and bias are f32.  Gradients do not depend on the order in which
    workgroups run.  First derivatives only."""
    if torch.is_grad_enabled() and (x.requires_grad or (weight is not None and weight.requires_grad) or
                                    (bias is not None and bias.requires_grad)):
        return _LayerNormFn.apply(x, weight, bias, eps, out_dtype)
    return ops.norm_fwd(x, weight, bias, eps, out_dtype, stats=False)[0].view(x.shape)
