"""Rotary positions for attention over voxels: pairs of a head's values turned by angles that grow with the
voxel's coordinates, queries and keys in one launch.

The reference has no counterpart; its networks would call torch for these.
"""
from __future__ import annotations

import functools
import math
import operator
from typing import Optional, Tuple

import torch
from torch.autograd import Function

from sparseconv import _native


class RotaryLayout:
    HALF = "half"
    INTERLEAVED = "interleaved"


class RotaryScaling:
    NONE = "none"
    LINEAR = "linear"
    NTK = "ntk"
    YARN = "yarn"


#: Full turns within the trained size below which YARN interpolates a pair wholly, and above which not at all.
YARN_TURNS = (1.0, 32.0)


def rotary_steps(pairs: int, base: float = 10000.0, scaling: str = RotaryScaling.NONE, factor: float = 1.0,
                 trained_size: Optional[int] = None) -> Tuple[Tuple[float, ...], float]:
    """(angle of one unit of position for each of an axis's pairs, amplitude of the rotation).

    Pair i's angle is ``base ** (-i / pairs)``, scaled for positions ``factor`` times as far as the trained
    ones: LINEAR divides it by the factor; NTK raises the base to ``base * factor ** (pairs / (pairs - 1))``, which
    divides the slowest pair's by the factor and leaves the fastest; YARN divides those that make less than
    one full turn within ``trained_size``, leaves those of more than 32, and goes linearly between them, with an
    amplitude of ``0.1 log(factor) + 1`` (on queries and keys, so scores grow by its square).
    """
    return _steps(operator.index(pairs), *_settings(base, scaling, factor, trained_size))


def _settings(base, scaling: str, factor, trained_size) -> tuple:
    """Their values now, by which plans are kept (a tensor of one may hold another at the next call)."""
    return (_native.constant("rotary positions", "base", base), scaling, _native.constant("rotary positions", "factor", factor),
            None if trained_size is None else _native.constant("rotary positions", "trained_size", trained_size))


@functools.lru_cache(maxsize=64)
def _steps(pairs: int, base: float, scaling: str, factor: float, trained_size: Optional[float]) -> Tuple[Tuple[float, ...], float]:
    if scaling not in (RotaryScaling.NONE, RotaryScaling.LINEAR, RotaryScaling.NTK, RotaryScaling.YARN):
        raise ValueError(f"unsupported scaling {scaling}")
    if not (base > 0.0 and math.isfinite(base)):
        raise ValueError(f"base must be positive and finite, got {base}")
    if not (factor >= 1.0 and math.isfinite(factor)):
        raise ValueError(f"factor must be at least 1 and finite, got {factor}")
    if scaling == RotaryScaling.NONE and factor != 1.0:
        raise ValueError("factor given without a scaling")
    if (scaling == RotaryScaling.YARN) != (trained_size is not None):
        raise ValueError("trained_size belongs to the yarn scaling, which needs it")
    if trained_size is not None and not trained_size > 0:
        raise ValueError(f"trained_size must be positive, got {trained_size}")
    if scaling == RotaryScaling.NTK and pairs > 1:
        base = base * factor ** (pairs / (pairs - 1))
    steps = [base ** (-i / pairs) for i in range(pairs)]
    if scaling == RotaryScaling.LINEAR:
        steps = [s / factor for s in steps]
    if scaling != RotaryScaling.YARN:
        return tuple(steps), 1.0
    low, high = YARN_TURNS
    for i, s in enumerate(steps):
        keep = min(1.0, max(0.0, (trained_size * s / (2.0 * math.pi) - low) / (high - low)))
        steps[i] = s * keep + s / factor * (1.0 - keep)
    return tuple(steps), 0.1 * math.log(factor) + 1.0


@functools.lru_cache(maxsize=64)
def _plan(size: int, rotary_dim: Optional[int], axes: int, layout: str, base: float, scaling: str, factor: float,
          trained_size: Optional[float]) -> _native.RotaryPlan:
    if rotary_dim is None:
        rotary_dim = size // 2 * 2
    pairs = rotary_dim // 2 // max(axes, 1)
    if rotary_dim % 2 or not 2 <= rotary_dim <= size or pairs < 1:
        raise ValueError(f"rotary_dim must be even, at most the head size {size} and at least twice the {axes} axes, "
                         f"got {rotary_dim}")
    return _native.RotaryPlan(layout, rotary_dim, axes, *_steps(pairs, base, scaling, factor, trained_size))


class SparseRotaryFunction(Function):
    @staticmethod
    def forward(ctx, query, key, positions, plan):
        ctx.save_for_backward(positions)
        ctx.plan = plan
        ctx.set_materialize_grads(False)
        turned = _native.rotary(query, key, positions, plan)
        constant = [t for t, needed in zip(turned, ctx.needs_input_grad) if t is not None and not needed]
        if constant:
            ctx.mark_non_differentiable(*constant)
        return turned

    @staticmethod
    def backward(ctx, grad_query, grad_key):
        """The same rotation backwards."""
        if torch.is_grad_enabled():              # create_graph=True: these gradients would be constants
            raise NotImplementedError("sparse_rotary has no second derivative")
        gq = grad_query if ctx.needs_input_grad[0] else None
        gk = grad_key if ctx.needs_input_grad[1] else None
        if gq is not None or gk is not None:
            gq, gk = _native.rotary(gq, gk, ctx.saved_tensors[0], ctx.plan, inverse=True)
        return gq, gk, None, None


def sparse_rotary(
    query: Optional[torch.Tensor],
    key: Optional[torch.Tensor],
    positions: torch.Tensor,
    layout: str = RotaryLayout.HALF,
    rotary_dim: Optional[int] = None,
    base: float = 10000.0,
    scaling: str = RotaryScaling.NONE,
    factor: float = 1.0,
    trained_size: Optional[int] = None,
) -> Tuple[Optional[torch.Tensor], Optional[torch.Tensor]]:
    """Queries and keys with their pairs (u, w) turned: (u cos - w sin, u sin + w cos) by the angle
    ``positions[row, axis] * step``.

    Args:
        query, key: [N, heads, D] and [N, key_heads, D] (fp32, fp16 or bf16, of one dtype) on CUDA, D <= 256. Rows
            and heads may be strided (a view into packed projections); a head's values that are not
            contiguous are copied first. Either may be None.
        positions: [N, axes] or [N] int32, any strides: ``x.indices[:, 1:]`` turns by the voxel's three
            coordinates, a serial number by one. Negative positions turn backwards.
        layout: ``RotaryLayout``: a pair is columns (i, i + rotary_dim / 2) (HALF) or (2 i, 2 i + 1) (INTERLEAVED).
        rotary_dim: columns of a head that hold pairs, even (None: all, but the last of an odd D). The axes
            take rotary_dim / 2 / axes pairs each, in order; pairs and columns left over are copied.
        base, scaling, factor, trained_size: angles per unit of position, see ``rotary_steps``.

    Returns:
        (query, key) turned, contiguous, rounded once from fp32; None for None. The fraction of a turn is computed
        in integers, exactly, so positions to the ends of int32 lose nothing.
    """
    _native.refuse_forward_mode("sparse_rotary", query, key)
    first = query if query is not None else key
    if first is None:
        raise ValueError("query or key is needed")
    if first.dim() != 3:
        raise ValueError(f"query and key must be [N, heads, D], got shape {list(first.shape)}")
    if positions.dim() not in (1, 2):
        raise ValueError(f"positions must be [N] or [N, axes], got shape {list(positions.shape)}")
    axes = 1 if positions.dim() == 1 else positions.shape[-1]
    plan = _plan(first.shape[2], None if rotary_dim is None else operator.index(rotary_dim), axes, layout,
                 *_settings(base, scaling, factor, trained_size))
    if torch.is_grad_enabled() and ((query is not None and query.requires_grad) or (key is not None and key.requires_grad)):
        return SparseRotaryFunction.apply(query, key, positions, plan)
    return _native.rotary(query, key, positions, plan)
