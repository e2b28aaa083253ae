"""Layer norm of a transformer block with its gradient, on the kernels of this package.

The block's norms in the reference are fp32 layer norms followed by the AdaLN modulation
(svoo/models/wan/custom_models.py:22-108); here norm, gain and offset are one pass over the tokens.
"""
from __future__ import annotations

from typing import Optional

import torch
from torch.autograd.function import once_differentiable

from . import ops


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, scale, shift, eps):
        y, mean, rstd = ops.layer_norm(x, weight, bias, scale, shift, eps, return_stats=True)
        ctx.save_for_backward(x, weight, scale, mean, rstd)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        x, weight, scale, mean, rstd = ctx.saved_tensors
        if grad.stride(-1) != 1 or grad.dim() > 3:
            grad = grad.contiguous()
        need = ctx.needs_input_grad
        dx, dgain, doffset = ops.layer_norm_backward(grad, x, mean, rstd, weight, scale, param_grads=any(need[1:5]))
        grads = (dx, dgain if need[1] else None, doffset if need[2] else None, dgain if need[3] else None,
                 doffset if need[4] else None)
        return grads + (None,)


def layer_norm(x: torch.Tensor, weight: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None,
               scale: Optional[torch.Tensor] = None, shift: Optional[torch.Tensor] = None, eps: float = 1e-6) -> torch.Tensor:
    """ops.layer_norm with gradients for x and the parameters (backward mode)."""
    ops.refuse_tangents(x, weight, bias, scale, shift)
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, weight, bias, scale, shift)):
        return _LayerNorm.apply(x, weight, bias, scale, shift, eps)
    return ops.layer_norm(x, weight, bias, scale, shift, eps)
