"""Global gradient norm over many tensors, and clipping by it, in two launches.

The reference has no counterpart; a training loop around it would call
``torch.nn.utils.clip_grad_norm_``, whose meaning ``clip_grad_norm_`` keeps.
"""
from __future__ import annotations

from typing import Iterable, Optional, Sequence, Union

import torch

from sparseconv import _native


def _norm_kind(norm_type: float) -> int:
    if norm_type == 2.0:
        return _native.CLIP_P2
    if norm_type == float("inf"):
        return _native.CLIP_INF
    raise ValueError(f"norm_type must be 2 or inf, got {norm_type}")


def clip_gradients(grads: Sequence[torch.Tensor], max_norm: float, norm_type: float = 2.0,
                   out: Optional[Sequence[torch.Tensor]] = None) -> torch.Tensor:
    """out[k] = grads[k] * min(1, max_norm / (total + 1e-6)), total the norm of all gradients as
    one vector.

    Args:
        grads: CUDA tensors of one device (fp32, fp16 or bf16, mixed freely), dense in memory. The
            list is not empty.
        max_norm: largest norm the result may have, >= 0.
        norm_type: 2.0 (square root of the sum of squares) or inf (largest magnitude).
        out: tensors of the gradients' sizes and dtypes, laid out alike; None clips in place. Outputs
            may not share memory with one another or with other gradients, so in place a tensor
            may not be listed twice.

    Returns:
        total: 0-dim fp32 tensor on the device (no synchronisation). If it is not finite the
        factor is the formula's (0 for inf, NaN for NaN): check it before taking the step.
    """
    grads = grads if isinstance(grads, (list, tuple)) else list(grads)
    if not grads:
        raise ValueError("no gradients given")
    if not max_norm >= 0.0:
        raise ValueError(f"max_norm must be >= 0, got {max_norm}")
    if out is not None and len(out) != len(grads):
        raise ValueError(f"{len(out)} outputs for {len(grads)} gradients")
    _native.refuse_forward_mode("clip_gradients", *grads, *(() if out is None else out))
    return _native.clip_gradients(grads, grads if out is None else out, max_norm, _norm_kind(norm_type))


def clip_grad_norm_(parameters: Union[torch.Tensor, Iterable[torch.Tensor]], max_norm: float,
                    norm_type: float = 2.0) -> torch.Tensor:
    """Clips the ``.grad`` of the parameters in place, as ``torch.nn.utils.clip_grad_norm_`` does,
    and returns their norm before clipping. Parameters without a gradient are passed over."""
    params = [parameters] if isinstance(parameters, torch.Tensor) else parameters
    grads = [p.grad for p in params if p.grad is not None]
    if not grads:
        _norm_kind(norm_type)
        return torch.tensor(0.0)
    return clip_gradients(grads, max_norm, norm_type)
