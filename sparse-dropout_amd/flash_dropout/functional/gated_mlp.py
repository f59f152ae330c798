"""A gated feed-forward block as one autograd function.

    forward   [G | U] = s (keep ⊙ X) W_in^T        H = act(G) ⊙ U        Y = s' (keep' ⊙ H) W_out^T
    backward  dH = s' (dY W_out) ⊙ keep'           dG = dH ⊙ U ⊙ act'(G)         dU = dH ⊙ act(G)
              dX = s ([dG | dU] W_in) ⊙ keep       dW_in = s [dG | dU]^T (keep ⊙ X)      dW_out = s' dY^T (keep' ⊙ H)

W_in [2 F, K] holds the gate's rows and behind them those of the other projection, so that both are one product.  act is SiLU,
GELU (erf form) or ReLU.  Sums and the gate are in 32 bits; G, U, H and dG, dU are rounded to the operands' type between the products,
whose operands they are.  G, U and H are kept for the backward; a forward that nothing is recorded of keeps none.
H is computed before G and U are rounded, so it may be finite where they are beyond their type (65504 in fp16) and kept as infinities.
Gradients then take the activation's limits: dG and dU are 0 behind a gate that is closed for all 32 bits, dG is dH U behind an open one;
dU is infinite where act(G) is not held, and dG where U is not.  (Where product and gate run apart, behind more than 131072 features, H is made
from G and U as they are kept.)

The reference has no gated block; arguments are those of the stack of layers (functional/blockwise_dropout_mlp_hip.py).
"""
from __future__ import annotations

import torch

from ..hip import _loader
from ..hip.binding_gemm import _block_size
from .blockwise_dropout_matmul_hip import draw_source
from .tracing import traceable

GATES = {"relu": 1, "gelu": 2, "silu": 3}  # enum sd_act


def _gate(activation) -> int:
    if activation not in GATES:
        raise ValueError(f"activation {activation!r}: a gate is one of {sorted(GATES)}")
    return GATES[activation]


@traceable
def gated_mlp(input: torch.Tensor, weight_in: torch.Tensor, weight_out: torch.Tensor, activation: str = "silu") -> torch.Tensor:
    """``(act(x W_g^T) * (x W_u^T)) W_out^T``: ``input`` [M, K], ``weight_in`` [2 F, K] (the rows of W_g, then those of W_u), ``weight_out``
    [N, F], all float16 or bfloat16 (under autocast: cast to its dtype).  Differentiable in all three.  Where nothing is recorded up to 64 rows may
    run in launches of their own, whose results differ in the last bits (up to 8 rows round the hidden activations to twice as many)."""
    return _loader.bridge().gated_mlp(input, weight_in, weight_out, 0, (0.0, 0.0), _gate(activation), None, None, None)


@traceable
def blockwise_dropout_gated_mlp(input: torch.Tensor, weight_in: torch.Tensor, weight_out: torch.Tensor, block_size, p,
                                activation: str = "silu", masks=None, seed: int | None = None) -> torch.Tensor:
    """:func:`gated_mlp` with blocks of the input and of the hidden activations dropped.  ``p``: a probability, or one for each of the two.
    ``masks``: a bool mask (True = dropped) or None for each of the two; None draws one, from ``seed`` (the second from ``seed + 1``) or the
    device-resident generator, a draw each.  Where p is 0 and no mask is given nothing is dropped and nothing drawn."""
    ps = (float(p), float(p)) if isinstance(p, (int, float)) else tuple(float(v) for v in p)
    if len(ps) != 2 or any(not 0 <= v < 1 for v in ps):
        raise ValueError("p must be one probability in [0, 1), or one for the input and one for the hidden activations")
    if masks is not None and len(masks) != 2:
        raise ValueError("masks are those of the input and of the hidden activations")
    draws = any(v > 0 and (masks is None or masks[i] is None) for i, v in enumerate(ps))
    return _loader.bridge().gated_mlp(input, weight_in, weight_out, _block_size(block_size), ps, _gate(activation),
                                      None if masks is None else list(masks), *(draw_source(input, seed) if draws else (None, None)))
