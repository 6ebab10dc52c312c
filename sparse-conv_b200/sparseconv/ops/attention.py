"""Attention over voxel features, within each sample of a batch: full, causal, over other rows (conditioning tokens,
pooling queries), in windows (a sample a window), with key heads shared by groups of query heads.

The reference has no counterpart; its networks would call torch for it.
"""
from __future__ import annotations

from typing import Optional

import torch
from torch.autograd import Function

from sparseconv import _native


class SparseAttentionFunction(Function):
    @staticmethod
    def forward(ctx, query, key, value, offsets, key_offsets, causal, scale):
        out, stats, ctx.args = _native.attention_forward(query, key, value, offsets, key_offsets, causal, scale, keep_stats=True)
        ctx.save_for_backward(query, key, value, offsets, key_offsets, out, stats)
        return out

    @staticmethod
    def backward(ctx, grad_out):
        """The probabilities again, from the inputs and what the forward kept."""
        if torch.is_grad_enabled():              # create_graph=True: these gradients would be constants
            raise NotImplementedError("sparse_attention has no second derivative")
        grads = _native.attention_backward_of(ctx.args, *ctx.saved_tensors, grad_out, ctx.needs_input_grad)
        return (*grads, None, None, None, None)


def sparse_attention(
    query: torch.Tensor,
    key: torch.Tensor,
    value: torch.Tensor,
    batch_offsets: Optional[torch.Tensor] = None,
    key_offsets: Optional[torch.Tensor] = None,
    causal: bool = False,
    scale: Optional[float] = None,
) -> torch.Tensor:
    """softmax(scale * query . key) value over the keys of each query's sample.

    Args:
        query: [N, heads, D] (fp32, fp16 or bf16) on CUDA, D <= 256. Rows and heads may be strided (views into packed
            projections); a head's values that are not contiguous are copied first.
        key, value: [Nk, key_heads, D] in the query's dtype; heads is a multiple of key_heads, and
            query head h reads key head h // (heads // key_heads).
        batch_offsets: [B + 1] int32 first query row of each sample (``SparseConvTensor.batch_offsets``); None: one
            sample. Attention in windows is a batch of windows: rows in window order, an offset a window.
        key_offsets: [B + 1] int32 first key row of each sample; None: ``batch_offsets``, with as many keys as
            queries. Offsets that do not ascend from 0 to the number of rows raise ``RuntimeError`` as the
            library's other device-side checks do. Samples may have no queries, or no keys.
        causal: each query sees the keys up to its own place, counted from the sample's end (the last query sees the
            last key), so one new query a sample sees everything. Keys that a query does not see leave its row and its
            gradient as they are, and it theirs, whatever they hold (NaN too).
        scale: factor of the scores, a positive number; None: D ** -0.5. It has no gradient.

    Returns:
        [N, heads, D] in the query's dtype; zeros for a query that sees no key. Scores, softmax and sums are fp32.
        fp16 and bf16 heads of up to 128 values run on the tensor cores, where the probabilities (and in the backward
        their gradients) enter the second product rounded to the dtype; fp32 and wider heads run in fp32 on the CUDA
        cores. For the backward a number a row is kept, and in 16 bits what out's rounding left out, as large as out. The
        gradients add in a fixed order: the same bits every run.
    """
    _native.refuse_forward_mode("sparse_attention", query, key, value)
    if batch_offsets is None and key_offsets is not None:
        raise ValueError("key_offsets given without batch_offsets")
    if key_offsets is None:
        if batch_offsets is not None and key.shape[0] != query.shape[0]:
            raise ValueError("as many keys as queries are needed where key_offsets is not given")
        key_offsets = batch_offsets
    scale = max(query.shape[-1], 1) ** -0.5 if scale is None else _native.constant("sparse_attention", "scale", scale)
    if torch.is_grad_enabled() and (query.requires_grad or key.requires_grad or value.requires_grad):
        return SparseAttentionFunction.apply(query, key, value, batch_offsets, key_offsets, bool(causal), scale)
    return _native.attention_forward(query, key, value, batch_offsets, key_offsets, causal, scale)[0]
