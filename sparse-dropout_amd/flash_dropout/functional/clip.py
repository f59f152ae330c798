"""The norm of many gradients together, and their clipping.

    norm = sqrt(Σ g²), or max |g|        c = min(1, max_norm / (norm + 1e-6))        g = c g

Squares are summed in 64 bits, in an order that the tensors' sizes fix: equal gradients have equal norms, a sum of squares neither overflows
nor vanishes where a gradient does not, and a norm beyond float32 is returned as infinity but clips by its own value.  A norm that is not
finite gives the factor that the formula gives, 0 or NaN, as torch's ``clip_grad_norm_`` does.
"""
from __future__ import annotations

import math
from collections.abc import Sequence

import torch

from ..hip import _loader
from .tracing import refused_under_trace

_NORMS = {2.0: 2, math.inf: 0}  # enum sd_norm


def _norm_type(norm_type) -> int:
    if float(norm_type) not in _NORMS:
        raise ValueError(f"norm_type must be 2 or inf (got {norm_type})")
    return _NORMS[float(norm_type)]


@refused_under_trace
def grad_norm(grads: Sequence[torch.Tensor], norm_type: float = 2.0, max_norm: float | None = None):
    """The norm of all ``grads`` (float16, bfloat16 or float32, also mixed, on one GPU) as a float32 on the GPU; with ``max_norm`` a pair of it
    and the factor that clips to ``max_norm``, for :func:`adamw_step`'s ``grad_scale``.  Nothing is written to the gradients."""
    norm, scale = _loader.bridge().grad_norm(list(grads), _norm_type(norm_type), None if max_norm is None else float(max_norm))
    return norm if max_norm is None else (norm, scale)


@refused_under_trace
def clip_grad_norm_(grads: Sequence[torch.Tensor], max_norm: float, norm_type: float = 2.0) -> torch.Tensor:
    """Scales ``grads`` (types as in :func:`grad_norm`, on one GPU) in place so that their norm is ``max_norm`` at most, and returns the norm they had.
    They must fill their memory and share none of it."""
    return _loader.bridge().clip_grads(list(grads), float(max_norm), _norm_type(norm_type))
