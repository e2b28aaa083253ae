"""Linear layers in 8-bit floating point: e4m3 operands with one scale per block of 128, sums in 32 bits.

Activations are quantised in every call in 1 x 128 blocks along the summed dimension, weights in 128 x 128 blocks: once, as
an Fp8Weight, for inference, or in every call from a higher-precision weight that is being trained.
"""
from __future__ import annotations

from typing import Optional, Union

import torch
import torch.nn as nn
from torch.autograd.function import once_differentiable

from . import ops
from .ops import Fp8Blocks as Fp8Weight


def _rows(x: torch.Tensor) -> torch.Tensor:
    """x [..., K] as a matrix with dense rows."""
    if x.dim() != 2:
        x = x.reshape(-1, x.shape[-1])
    return x if x.shape[1] == 1 or x.stride(1) == 1 else x.contiguous()


class _Trained(torch.autograd.Function):
    """A weight that is quantised in the call: one call of the library forward, one backward."""

    @staticmethod
    def forward(ctx, x, weight, bias):
        ctx.kept = ctx.needs_input_grad[:2]
        ctx.dtypes = weight.dtype, None if bias is None else bias.dtype
        ctx.shape = weight.shape
        y, saved = ops.linear_train_forward(x, weight, bias, *ctx.kept)
        ctx.save_for_backward(saved)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        need_x, need_w, need_b = ctx.needs_input_grad
        saved, = ctx.saved_tensors
        return ops.linear_train_backward(_rows(grad), saved, ctx.shape[1], *ctx.kept, need_x, ctx.dtypes[0] if need_w else None,
                                         ctx.dtypes[1] if need_b else None)


class _Stored(torch.autograd.Function):
    """A weight that is a constant."""

    @staticmethod
    def forward(ctx, x, weight, bias):
        ctx.bias_dtype = None if bias is None else bias.dtype
        if ctx.needs_input_grad[0]:
            w = weight.transposed()                         # raises without one
            ctx.save_for_backward(w.q, w.scale)
        return ops.mm_fp8(ops.quantize_rows(x), weight, bias, None, x.dtype)

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        grad = _rows(grad)
        dx = db = None
        if ctx.needs_input_grad[0]:
            dx = ops.mm_fp8(ops.quantize_rows(grad), Fp8Weight(*ctx.saved_tensors), None, None, grad.dtype)
        if ctx.needs_input_grad[2]:
            db = ops.quantize_columns(grad, ctx.bias_dtype)[1] if grad.shape[0] else grad.new_zeros(grad.shape[1], dtype=ctx.bias_dtype)
        return dx, None, db


class _NoRows(torch.autograd.Function):
    """A trained layer without rows: an empty result, gradients of zeros."""

    @staticmethod
    def forward(ctx, x, weight, bias):
        ctx.like = [None if t is None else (t.shape, t.dtype) for t in (x, weight, bias)]
        return x.new_empty((0, weight.shape[0]))

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        return tuple(grad.new_zeros(like[0], dtype=like[1]) if need else None for like, need in zip(ctx.like, ctx.needs_input_grad))


def check_status(device: torch.device) -> None:
    """Raises if a layer norm or an 8-bit product on this device has given up on one of its bounded waits (its output is then
    incomplete).  Reads a device word, so it synchronises: call it once per step or at the end of a run."""
    if ops.linear_status(device) != 0:
        raise RuntimeError(f"a layer norm or an 8-bit product on {device} timed out on a barrier; output incomplete")


def linear_fp8(x: torch.Tensor, weight: Union[torch.Tensor, Fp8Weight], bias: Optional[torch.Tensor] = None,
               activation: Optional[str] = None) -> torch.Tensor:
    """act(x weight^T + bias) for x [..., K] (bf16, fp16 or fp32) -> [..., N] of x's type.  `weight` is an Fp8Weight, or a tensor
    [N, K] that is quantised in the call.  Gradients flow to x, to a weight that is a tensor and to bias, through
    products in e4m3 as well: the gradient of the output is quantised in blocks along what each of them sums over, and
    rounding counts as the identity.  An Fp8Weight is a constant; with it the gradient of x needs its transpose
    (ops.quantize_blocks(w, transposed=True)).  An activation has no gradient here."""
    ops.refuse_tangents(x, weight if isinstance(weight, torch.Tensor) else None, bias)
    training = torch.is_grad_enabled() and (x.requires_grad or (isinstance(weight, torch.Tensor) and weight.requires_grad) or
                                            (bias is not None and bias.requires_grad))
    m = _rows(x)
    if training:
        if activation is not None:
            raise ValueError("linear_fp8 has no gradient through an activation: apply it to the result")
        trained = isinstance(weight, torch.Tensor)
        y = (_Stored if not trained else _Trained if m.shape[0] else _NoRows).apply(m, weight, bias)
    else:
        w = ops.quantize_blocks(weight) if isinstance(weight, torch.Tensor) else weight
        y = ops.linear_fp8(m, w, bias, activation)
    return y if x.dim() == 2 else y.view(*x.shape[:-1], y.shape[1])


def mlp_fp8(x: torch.Tensor, w1: Fp8Weight, bias1: Optional[torch.Tensor], w2: Fp8Weight,
            bias2: Optional[torch.Tensor]) -> torch.Tensor:
    """linear(gelu(linear(x, w1, bias1)), w2, bias2), GELU with its tanh formula: the feed-forward of a block.  The hidden rows are
    quantised from their 32-bit values as the first product leaves its registers.  Inference only."""
    ops.refuse_tangents(x, bias1, bias2)
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, bias1, bias2)):
        raise ValueError("mlp_fp8 has no gradient: use two linear_fp8 around the activation")
    h = ops.linear_fp8(_rows(x), w1, bias1, "gelu", ops.E4M3)
    y = ops.mm_fp8(h, w2, bias2, None, x.dtype)
    return y if x.dim() == 2 else y.view(*x.shape[:-1], y.shape[1])


class Fp8Linear(nn.Module):
    """An nn.Linear for inference whose weight is held in e4m3, one byte per number: forward is linear_fp8 with the bias and
    type of the input.  The bytes and scales are kept as uint8 buffers, which follow the module to a device and through a
    state dict, and which a cast of the module's floating-point type leaves alone."""

    def __init__(self, in_features: int, out_features: int, bias: bool = True, input_grad: bool = False, device=None,
                 dtype: Optional[torch.dtype] = None):
        super().__init__()
        self.in_features, self.out_features = in_features, out_features
        blocks = ((out_features + 127) // 128, (in_features + 127) // 128)

        def buffer(rows, columns):
            return torch.zeros(rows, columns, dtype=torch.uint8, device=device)

        self.register_buffer("weight_q", buffer(out_features, ops._pad16(in_features)))
        self.register_buffer("weight_scale", buffer(blocks[0], 4 * blocks[1]))
        self.register_buffer("weight_qt", buffer(in_features, ops._pad16(out_features)) if input_grad else None)
        self.bias = nn.Parameter(torch.zeros(out_features, device=device, dtype=dtype), requires_grad=False) if bias else None

    @classmethod
    def from_linear(cls, linear: nn.Linear, input_grad: bool = False) -> "Fp8Linear":
        """Quantises the weight of a linear layer on its GPU.  input_grad keeps the transpose too, for the gradient of the input."""
        w = linear.weight.detach()
        m = cls(linear.in_features, linear.out_features, linear.bias is not None, input_grad, w.device, w.dtype)
        m.set_weight(ops.quantize_blocks(w, transposed=input_grad))
        if linear.bias is not None:
            m.bias.data.copy_(linear.bias.detach())
        return m.train(linear.training)

    @torch.no_grad()
    def set_weight(self, w: Fp8Weight) -> None:
        N, K = w.shape
        if (N, K) != (self.out_features, self.in_features):
            raise ValueError(f"expected a weight [{self.out_features}, {self.in_features}], got {[N, K]}")
        self.weight_q[:, :K].copy_(w.q.view(torch.uint8))
        self.weight_scale.copy_(w.scale.contiguous().view(torch.uint8))
        if self.weight_qt is not None:
            self.weight_qt[:, :N].copy_(w.transposed().q.view(torch.uint8))

    @property
    def weight(self) -> Fp8Weight:
        qt = None if self.weight_qt is None else self.weight_qt.view(ops.E4M3)[:, :self.out_features]
        return Fp8Weight(self.weight_q.view(ops.E4M3)[:, :self.in_features], self.weight_scale.view(torch.float32), qt)

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        return linear_fp8(x, self.weight, self.bias)

    def extra_repr(self) -> str:
        return f"in_features={self.in_features}, out_features={self.out_features}, bias={self.bias is not None}"


class Fp8FeedForward(nn.Module):
    """Linear, GELU (tanh formula), Linear on e4m3 weights, for inference: forward is mlp_fp8."""

    def __init__(self, first: Fp8Linear, second: Fp8Linear):
        super().__init__()
        self.first, self.second = first, second

    @classmethod
    def from_sequential(cls, seq: nn.Sequential) -> "Fp8FeedForward":
        if len(seq) != 3 or not isinstance(seq[0], nn.Linear) or not isinstance(seq[2], nn.Linear) or \
                not isinstance(seq[1], nn.GELU) or seq[1].approximate != "tanh":
            raise ValueError("expected Linear, GELU(approximate='tanh'), Linear")
        return cls(Fp8Linear.from_linear(seq[0]), Fp8Linear.from_linear(seq[2]))

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        return mlp_fp8(x, self.first.weight, self.first.bias, self.second.weight, self.second.bias)
