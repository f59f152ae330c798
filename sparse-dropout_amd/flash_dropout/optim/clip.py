"""``clip_grad_norm_`` with the arguments of ``torch.nn.utils.clip_grad_norm_``, two launches for each 176 parameters.

Narrower than torch's in what it takes: ``norm_type`` 2 or inf, dense gradients in float16, bfloat16 or float32 (also mixed) that are all on one GPU, fill
their memory and share none of it, and no negative ``max_norm``.  Everything else raises."""
from __future__ import annotations

import torch

from ..functional.clip import clip_grad_norm_ as clip_gradients
from ..functional.clip import grad_norm


@torch.no_grad()
def clip_grad_norm_(parameters, max_norm: float, norm_type: float = 2.0, error_if_nonfinite: bool = False,
                    foreach: bool | None = None) -> torch.Tensor:
    """Clips the gradients of ``parameters`` (an iterable of tensors, or one) to a joint norm of ``max_norm`` and returns the norm they had.
    Parameters without a gradient are left out; what is refused is named above.  ``error_if_nonfinite`` waits for the norm, and then leaves the gradients as they are where it is
    not finite and raises; without it nothing waits.  ``foreach`` is taken for the sake of calls that give it: there is one way here."""
    grads = [p.grad for p in ([parameters] if isinstance(parameters, torch.Tensor) else parameters) if p.grad is not None]
    if not grads:
        return torch.tensor(0.0)
    if error_if_nonfinite and not torch.isfinite(grad_norm(grads, norm_type)):
        raise RuntimeError(f"the norm of order {float(norm_type)} of the gradients is not finite: they cannot be clipped")
    return clip_gradients(grads, max_norm, norm_type)
