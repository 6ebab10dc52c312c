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


def _bias(bias: Optional[torch.Tensor], dtype: torch.dtype) -> Optional[torch.Tensor]:
    """As the kernels add it: the features' dtype, or fp32 for every other."""
    return bias if bias is None or bias.dtype == dtype else bias.to(torch.float32)


class SparseLinearFunction(Function):
    @staticmethod
    def forward(ctx, feats, weight, bias, residual, activation):
        w = weight.to(feats.dtype).contiguous()
        b = _bias(bias, feats.dtype)
        needs = ctx.needs_input_grad
        keep = activation != Activation.NONE and (needs[0] or needs[1] or needs[2])
        out, preact = _native.linear_forward(feats, w, b, residual, activation, keep_preact=keep)
        ctx.save_for_backward(feats, w, preact)
        ctx.settings = (_native.ACTIVATIONS[activation], weight.dtype, None if bias is None else bias.dtype)
        return out

    @staticmethod
    def backward(ctx, grad_out):
        if torch.is_grad_enabled():              # create_graph=True: these gradients would be constants
            raise NotImplementedError("sparse_linear has no second derivative")
        feats, weight, preact = ctx.saved_tensors
        needs = ctx.needs_input_grad
        if not grad_out.is_contiguous():
            grad_out = grad_out.contiguous()
        grads = (None, None, None)
        if needs[0] or needs[1] or needs[2]:
            grads = _native.linear_backward_of(grad_out, preact, feats, weight, *ctx.settings, needs)
        return (*grads, grad_out if needs[3] else None, None)


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
        bias: [Co] bias in the feature dtype or fp32, added in fp32 (others are cast to fp32), or None.
        residual: [N, Co] added after the activation, in the feature dtype, contiguous, or None.
        activation: any ``Activation`` value; GELU is the exact one (normal distribution function).

    Returns:
        [N, Co] in the feature dtype: fp32 accumulation and epilogue, rounded once. fp16 and bf16
        run on the tensor cores where the channel counts are multiples of 8 and the tensors start
        on 16-byte boundaries, or where copies into whole rows of 8 pay; everything else in fp32 on the
        CUDA cores. For the backward of an activation its argument is kept in the feature
        dtype, and the gradient at it is rounded to the feature dtype before the products (bf16
        gradients are then off by 2.4e-3 of their norm, 1.7e-3 of which any bf16 result is); weight and
        bias gradients come in the parameters' dtypes, summed in fp32 in a fixed order.
    """
    _native.refuse_forward_mode("sparse_linear", feats, weight, bias, residual)
    if torch.is_grad_enabled() and (feats.requires_grad or weight.requires_grad or
                                    (bias is not None and bias.requires_grad) or
                                    (residual is not None and residual.requires_grad)):
        return SparseLinearFunction.apply(feats, weight, bias, residual, activation)
    return _native.linear_forward(feats, weight.to(feats.dtype), _bias(bias, feats.dtype), residual, activation)[0]
