"""LayerNorm over rows of any width up to 16384 in f32, bf16 or fp16, as a differentiable function: for norms of
models built around the Performer stack, where the stack's own kernels (ops.ln_fwd / ln_bwd: f32 residual stream, at most 256
columns) do not apply.  The package's own modules do not call it: StudentEncoder and scMomer keep torch's nn.LayerNorm.
"""
from __future__ import annotations

from typing import Optional

import torch

from . import _lib


def layer_norm(x: torch.Tensor, weight: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None,
               eps: float = 1e-5, *, out_dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """(x - mean) / sqrt(var + eps) * weight + bias over the last dimension D of x [..., D].

    x: f32, bf16 or fp16 on the GPU, 1 <= D <= 16384, any row stride (other layouts are copied first); weight, bias:
    f32 [D] or None (1, 0).  The result has x's type, or bfloat16 from f32 with ``out_dtype=torch.bfloat16``;
    statistics and the gradients of weight and bias are f32.  Results do not depend on the order in which workgroups
    run; a row's last place may depend on the number of rows in the call.

    First derivatives only, in reverse mode: under forward-mode differentiation, a tracer (torch.jit.trace, make_fx),
    torch.func's transforms or with tensor subclasses that have a dispatch of their own it raises NotImplementedError.  A
    backward pass under capture into a graph is refused while an eager graph on the default stream holds a leaf that it reaches (its gradient would
    have to join that stream)."""
    return _lib.torch_ops.layer_norm(x, weight, bias, eps, out_dtype)
