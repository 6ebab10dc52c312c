"""Pointwise (1x1x1) linear layer over voxel features, with bias, activation and residual in the
product's epilogue: the layer between submanifold convolutions that needs no neighbour map.

The reference has no counterpart; its networks would call torch for this layer.
"""
from __future__ import annotations

from typing import Optional

import torch
from torch.autograd import Function

from sparseconv import _native


class Activation:
    NONE = "none"
    RELU = "relu"
    GELU = "gelu"
    SILU = "silu"


class SparseLinearFunction(Function):
    @staticmethod
    def forward(ctx, feats, weight, bias, residual, activation):
        w = weight.to(feats.dtype)
        b = None if bias is None else bias.to(feats.dtype)
        keep = activation != Activation.NONE and any(ctx.needs_input_grad[:3])
        out, preact = _native.linear_forward(feats, w, b, residual, activation, keep_preact=keep)
        ctx.save_for_backward(feats, w, preact)
        ctx.dtypes = (weight.dtype, None if bias is None else bias.dtype)
        ctx.activation = activation
        return out

    @staticmethod
    def backward(ctx, grad_out):
        feats, weight, preact = ctx.saved_tensors
        weight_dtype, bias_dtype = ctx.dtypes
        grad_out = grad_out.to(feats.dtype).contiguous()
        grad_feats = grad_weight = grad_bias = None
        if any(ctx.needs_input_grad[:3]):
            grad_feats, grad_weight, grad_bias = _native.linear_backward(
                grad_out, preact, feats, weight, ctx.activation, weight_dtype, bias_dtype, ctx.needs_input_grad[:3])
        return grad_feats, grad_weight, grad_bias, grad_out if ctx.needs_input_grad[3] else None, None


def sparse_linear(
    feats: torch.Tensor,
    weight: torch.Tensor,
    bias: Optional[torch.Tensor] = None,
    residual: Optional[torch.Tensor] = None,
    activation: str = Activation.NONE,
) -> torch.Tensor:
    """residual + activation(feats @ weight.T + bias)

    Args:
        feats: [N, C] input features (fp32, fp16 or bf16), contiguous, on CUDA.
        weight: [Co, C] weights (cast to the feature dtype).
        bias: [Co] bias or None (cast to the feature dtype).
        residual: [N, Co] added after the activation, in the feature dtype, contiguous, or None.
        activation: any ``Activation`` value; GELU is the exact one (normal distribution function).

    Returns:
        [N, Co] in the feature dtype: fp32 accumulation and epilogue, rounded once. fp16 and bf16
        with channel counts that are multiples of 8 run on the tensor cores, everything else in
        fp32 on the CUDA cores. For the backward of an activation the product (before the
        activation) is kept in the feature dtype; weight and bias gradients come in the
        parameters' dtypes, summed in fp32 in a fixed order.
    """
    if not torch.is_grad_enabled() or not any(
            t is not None and t.requires_grad for t in (feats, weight, bias, residual)):
        return _native.linear_forward(feats, weight.to(feats.dtype), None if bias is None else bias.to(feats.dtype),
                                      residual, activation)[0]
    return SparseLinearFunction.apply(feats, weight, bias, residual, activation)
