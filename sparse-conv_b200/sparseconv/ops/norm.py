"""Norms over voxel features, and the gated residual step between two blocks with a norm on
either side of it, as one pass over the features.

The reference has no counterpart; its networks would call torch for these.
"""
from __future__ import annotations

from typing import Optional, Tuple

import torch
from torch.autograd import Function

from sparseconv import _native


class Norm:
    NONE = "none"
    LAYER = "layer"
    RMS = "rms"


class ResidualNormFunction(Function):
    @staticmethod
    def forward(ctx, feats, residual, gate, weight, bias, next_weight, next_bias, batch_offsets,
                residual_scale, norm, next_norm, eps):
        params = (gate, weight, bias, next_weight, next_bias)
        hidden, normed, stats, ctx.args = _native.residual_norm_forward(
            feats, residual, params, batch_offsets, residual_scale, norm, next_norm, eps, keep_stats=True)
        ctx.save_for_backward(feats, residual, *params, batch_offsets, stats)
        ctx.set_materialize_grads(False)
        return hidden, normed

    @staticmethod
    def backward(ctx, grad_hidden, grad_normed):
        """From the inputs, recomputed in fp32, and the forward's row statistics (16 bytes a row)."""
        if torch.is_grad_enabled():              # create_graph=True: these gradients would be constants
            raise NotImplementedError("sparse_residual_norm has no second derivative")
        if grad_hidden is None and grad_normed is None:
            return (None,) * 12
        feats, residual, *params, batch_offsets, stats = ctx.saved_tensors
        gh, gn = (g if g is None or g.is_contiguous() else g.contiguous() for g in (grad_hidden, grad_normed))
        grads = _native.residual_norm_backward_of(
            ctx.args, feats, residual, params, batch_offsets, stats, gh, gn, ctx.needs_input_grad)
        return (*grads, None, None, None, None, None)


def sparse_residual_norm(
    feats: torch.Tensor,
    residual: Optional[torch.Tensor] = None,
    gate: Optional[torch.Tensor] = None,
    batch_offsets: Optional[torch.Tensor] = None,
    residual_scale: float = 1.0,
    norm: str = Norm.NONE,
    weight: Optional[torch.Tensor] = None,
    bias: Optional[torch.Tensor] = None,
    next_norm: str = Norm.LAYER,
    next_weight: Optional[torch.Tensor] = None,
    next_bias: Optional[torch.Tensor] = None,
    eps: float = 1e-5,
) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """The step from one block's output to the next block's input:

        hidden = residual_scale * residual + gate * (norm(feats) * weight + bias)
        normed = next_norm(hidden) * next_weight + next_bias

    Args:
        feats: [N, C] output of a block (fp32, fp16 or bf16), contiguous, on CUDA; C <= 8192.
        residual: [N, C] the features that went into the block, in the same dtype, or None.
        gate, weight, bias, next_weight, next_bias: [C], or [B, C] with a row for each sample of
            the batch, in fp32 or the features' dtype, contiguous; None for 1 (gate and weights)
            or 0 (biases).
        batch_offsets: [B + 1] int32 first row of each sample (``SparseConvTensor.batch_offsets``),
            needed when a parameter has a row per sample. Offsets that do not ascend from 0 to N
            raise ``RuntimeError`` as the library's other device-side checks do.
        residual_scale: factor of the residual.
        norm: ``Norm`` of the block's output (``Norm.NONE``: taken as it is).
        next_norm: ``Norm`` before the next block (``Norm.NONE``: ``normed`` is None).
        eps: added to the variance (LAYER) or the mean square (RMS).

    Returns:
        (hidden [N, C], normed [N, C] or None) in the features' dtype; statistics and products are
        fp32 and ``normed`` is computed from ``hidden`` before that is rounded.
    """
    params = (feats, residual, gate, weight, bias, next_weight, next_bias)
    _native.refuse_forward_mode("sparse_residual_norm", *params)
    if not torch.is_grad_enabled() or not any(t is not None and t.requires_grad for t in params):
        return _native.residual_norm_forward(feats, residual, params[2:], batch_offsets, residual_scale,
                                             norm, next_norm, eps)
    return ResidualNormFunction.apply(*params, batch_offsets, residual_scale, norm, next_norm, eps)


def sparse_norm(
    feats: torch.Tensor,
    weight: Optional[torch.Tensor] = None,
    bias: Optional[torch.Tensor] = None,
    batch_offsets: Optional[torch.Tensor] = None,
    norm: str = Norm.LAYER,
    eps: float = 1e-5,
) -> torch.Tensor:
    """norm(feats) * weight + bias over the channels of each voxel: ``sparse_residual_norm``
    without gate, residual and following norm; arguments as there."""
    return sparse_residual_norm(feats, batch_offsets=batch_offsets, norm=norm, weight=weight, bias=bias,
                                next_norm=Norm.NONE, eps=eps)[0]
