"""One AdamW step over many tensors, the two averages held in 32 or in 8 bits.

    t = step + 1        m = β1 m + (1 - β1) g        v = β2 v + (1 - β2) g²
    p = p (1 - lr·decay) - lr / (1 - β1^t) · m / (sqrt(v / (1 - β2^t)) + eps)

Averages in 8 bits are codes, a byte an element in the order of the parameter's memory, and a power of two for each 128 of them
(uint8, its exponent plus 127): for m e4m3, whose largest number is 448; for v, which has no sign, five bits of exponent
(bias 15) and three of mantissa, the largest 61440.  The scale is the least with which the block stays within the largest
number.  Both are rounded at random, up with the probability that the value's place between two codes says: an average moves by a
thousandth of its distance in a step, and rounded to nearest it would stay where it is.  The random bits are a function of t
and the element's index (M. O'Neill's permuted congruential generator), so equal runs have equal states: elements of one index in
different tensors, and both averages of an element, are rounded by parts of one word.  Zeros are codes 0 with scales 127.

The update is computed in 32 bits.  With averages in 8 bits, which are computed in 64, its root and reciprocal are the hardware's, one unit of
the last place off, not the exact ones that it has with averages in 32 bits.
"""
from __future__ import annotations

from collections.abc import Sequence

import torch

from ..hip import _loader
from .tracing import refused_under_trace

STATE_BLOCK = 128  # elements of a state in 8 bits that share a scale


def _split(averages, name):
    """(tensors, scales): scales empty for averages in 32 bits."""
    averages = list(averages)
    pairs = [isinstance(a, (tuple, list)) for a in averages]
    if not any(pairs):
        return averages, []
    if not all(pairs) or any(len(a) != 2 for a in averages):
        raise ValueError(f"{name} must be float32 tensors, or a (codes, scales) pair each")
    return [a[0] for a in averages], [a[1] for a in averages]


@refused_under_trace
def adamw_step(params: Sequence[torch.Tensor], grads: Sequence[torch.Tensor], exp_avgs: Sequence, exp_avg_sqs: Sequence,
               step: torch.Tensor, *, lr: float | torch.Tensor = 1e-3, betas: tuple[float, float] = (0.9, 0.999), eps: float = 1e-8,
               weight_decay: float = 1e-2, grad_scale: torch.Tensor | None = None) -> None:
    """Updates ``params`` (float16, bfloat16 or float32, also mixed), both averages and ``step`` in place.  The averages are float32
    tensors laid out like their parameters or ``(codes, scales)`` pairs of uint8 tensors, the codes laid out like their parameters too or in one
    run.  ``step``: one int64 on the GPU, the number of steps so far, moved on by the call itself: a captured graph counts its replays.
    ``lr`` may be a float32 tensor on the GPU, which a captured graph reads at every replay, and so may ``grad_scale``, which gradients are
    multiplied by as they are read (:func:`grad_norm` gives the one that clips).  None of these lies in what is written.  One launch for each 56 tensors of a dtype.
    ``torch.jit.trace`` is refused."""
    beta1, beta2 = (float(b) for b in betas)
    firsts, first_scales = _split(exp_avgs, "exp_avgs")
    seconds, second_scales = _split(exp_avg_sqs, "exp_avg_sqs")
    if bool(first_scales) != bool(second_scales):
        raise ValueError("both averages are held in 32 bits, or both in 8")
    at = lr if isinstance(lr, torch.Tensor) else None
    _loader.bridge().adamw_step(list(params), list(grads), firsts, seconds, first_scales, second_scales, step, at,
                                0.0 if at is not None else float(lr), beta1, beta2, float(eps), float(weight_decay), grad_scale)


@refused_under_trace
def adamw_state_values(exp_avgs: Sequence, exp_avg_sqs: Sequence) -> tuple[list[torch.Tensor], list[torch.Tensor]]:
    """Averages in 8 bits, ``(codes, scales)`` pairs, as float32 tensors laid out like the codes, in one launch for each 56 of them."""
    firsts, first_scales = _split(exp_avgs, "exp_avgs")
    seconds, second_scales = _split(exp_avg_sqs, "exp_avg_sqs")
    if len(first_scales) != len(firsts) or len(second_scales) != len(seconds):
        raise ValueError("averages in 8 bits are (codes, scales) pairs")
    values = _loader.bridge().adamw_state_values([*firsts, *seconds], [*first_scales, *second_scales],
                                                 [0] * len(firsts) + [1] * len(seconds))
    return values[:len(firsts)], values[len(firsts):]


def adamw_empty_state(param: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """A ``(codes, scales)`` pair of zeros for one average of ``param``, the codes laid out like it."""
    return (torch.zeros_like(param, dtype=torch.uint8, memory_format=torch.preserve_format),
            torch.full((-(-param.numel() // STATE_BLOCK),), 127, dtype=torch.uint8, device=param.device))
