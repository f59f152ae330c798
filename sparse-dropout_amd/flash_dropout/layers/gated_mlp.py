"""``GatedMLP``: a bias-free gated feed-forward block with dropout on the inputs of its products.

The reference's feed-forward block is ``DropoutMM``, an activation, ``DropoutMM`` (eval/llm/model.py:58-66); here the activation of one
projection multiplies another.  Variants and arguments are those of ``DropoutMM`` (layers/dropout_mm.py)."""
from __future__ import annotations

import math

import torch
from torch import nn

from .. import functional as F

VARIANTS = ("none", "vanilla", "blockwise[naive]", "blockwise[hip]")
_ACTIVATIONS = {"relu": nn.functional.relu, "gelu": nn.functional.gelu, "silu": nn.functional.silu}


class GatedMLP(nn.Module):
    """``y = dropout(act(g) * u) @ W_out.T`` with ``[g | u] = dropout(x) @ W_in.T``: ``weight_in`` [2 hidden, in] (the gate's rows first),
    ``weight_out`` [out, hidden], no biases.

    ``variant``: "none" (no dropout), "vanilla" (element-wise dropout), "blockwise[naive]" or "blockwise[hip]", which need ``block_size=``.
    In eval mode nothing is dropped; "blockwise[hip]" is then the same kernels without masks, the others are torch's operations.  Leading
    dimensions are flattened first, as in ``DropoutMM``."""

    __constants__ = ["in_features", "hidden_features", "out_features"]

    def __init__(self, in_features: int, hidden_features: int, out_features: int | None = None, p: float = 0.1, variant: str = "vanilla",
                 activation: str = "silu", **kwargs) -> None:
        super().__init__()
        if activation not in _ACTIVATIONS:
            raise ValueError(f"activation {activation!r}: a gate is one of {sorted(_ACTIVATIONS)}")
        self.in_features = in_features
        self.hidden_features = hidden_features
        self.out_features = in_features if out_features is None else out_features
        self.p = p
        self.variant = variant
        self.activation = activation
        self.kwargs = kwargs
        self.weight_in = nn.Parameter(torch.empty(2 * hidden_features, in_features))
        self.weight_out = nn.Parameter(torch.empty(self.out_features, hidden_features))
        self.reset_parameters()

    def reset_parameters(self) -> None:
        # as DropoutMM initialises each of the three matrices
        nn.init.kaiming_uniform_(self.weight_in, a=math.sqrt(5))
        nn.init.kaiming_uniform_(self.weight_out, a=math.sqrt(5))

    def forward(self, input: torch.Tensor) -> torch.Tensor:
        x = input.reshape(-1, input.shape[-1])
        v = self.variant
        if v == "blockwise[hip]":
            if self.training:
                y = F.hip_blockwise_dropout_gated_mlp(x, self.weight_in, self.weight_out, self.kwargs["block_size"], self.p, self.activation)
            else:
                y = F.gated_mlp(x, self.weight_in, self.weight_out, self.activation)
        else:
            if v == "none" or (not self.training and v in VARIANTS):
                product = nn.functional.linear
            elif v == "vanilla":
                product = lambda a, w: F.vanilla_dropout_matmul(a, w, self.p)
            elif v == "blockwise[naive]":
                product = lambda a, w: F.naive_blockwise_dropout_matmul(a, w, self.kwargs["block_size"], self.p)
            else:
                raise ValueError(f"Unknown variant {self.variant}")
            gate, up = product(x, self.weight_in).chunk(2, dim=-1)
            y = product(_ACTIVATIONS[self.activation](gate) * up, self.weight_out)
        return y.reshape(*input.shape[:-1], self.out_features)

    def extra_repr(self) -> str:
        return (f"in_features={self.in_features}, hidden_features={self.hidden_features}, out_features={self.out_features}, p={self.p}, "
                f"variant={self.variant!r}, activation={self.activation!r}")
