"""Linear layers in 8-bit floating point with a scale for each block of 128.

A matrix in 8 bits is two tensors: e4m3 codes [rows, columns filled up with zeros to a multiple of 128] and powers of two
(``torch.float8_e8m0fnu``), one for each block of 1 x 128 (``scales`` [rows, blocks]) or of 128 x 128 (``scales``
[ceil(rows / 128), blocks]).  A block's scale is the least power of two with which its largest finite magnitude stays within 448, the
largest number of e4m3; it divides without rounding, so a value is rounded once, by at most half of the 2^-3 between two
codes.  What is not finite becomes NaN; a value below 2^-10 of its block's scale becomes zero.

    serving     y  = q(x) q(W)^T                       x in 1 x 128 blocks, quantized by the call; W kept in 128 x 128 blocks
    training    Y  = s (keep ⊙ q(X)) q(W)^T            X in 1 x 128, W in 128 x 128 blocks
                dX = s (q(dY) q(W)) ⊙ keep             dY in 1 x 128 blocks; W's 128 x 128 blocks read the other way
                dW = s q'(dY)^T (keep ⊙ q'(X))         both in 128 x 1 blocks: this sum runs over the tokens

with s = 1 / (1 - p), sums in fp32 and one rounding to the operands' dtype.  The gradients are those of the quantized matrices (the
quantizer passes gradients through).  Blocks of the dropout mask are multiples of 128, so a dropped block is neither quantized nor
multiplied.  The reference has no 8-bit path; the linear layer has the arguments of its block-dropout matmul
(functional/blockwise_dropout_matmul_cuda.py:56-59) and of the naive one with the mask given (functional/naive.py:8-14).
"""
from __future__ import annotations

import torch

from ..hip import _loader
from ..hip.binding_gemm import _block_size
from .blockwise_dropout_matmul_hip import draw_source
from .tracing import _RecordedConstantCall, _RecordedPlainCall, traceable


@traceable(recorded=_RecordedConstantCall, cast=False)
def fp8_quantize(x: torch.Tensor, block=(1, 128)) -> tuple[torch.Tensor, torch.Tensor]:
    """(codes, scales) of a float16, bfloat16 or float32 matrix, in blocks of (1, 128) or (128, 128).  The scales of (1, 128)
    blocks lie one 128-block's after the other in memory (strides (1, n)), as the products read them.  They carry no gradient."""
    block = tuple(block)
    if block not in ((1, 128), (128, 128)):
        raise ValueError(f"block must be (1, 128) or (128, 128), got {block}")
    return _loader.bridge().fp8_quantize(x, block[0])


@traceable(recorded=_RecordedConstantCall, cast=False)
def fp8_dequantize(data: torch.Tensor, scales: torch.Tensor, cols: int | None = None,
                   dtype: torch.dtype = torch.float32) -> torch.Tensor:
    """The values of codes and scales as ``dtype``: the first ``cols`` columns (default: all, the zeros behind the last too),
    without a gradient."""
    # (an extent that a trace takes off a tensor is a tensor itself)
    return _loader.bridge().fp8_dequantize(data, scales, int(cols) if isinstance(cols, torch.Tensor) else cols, dtype)


@traceable(recorded=_RecordedPlainCall)
def fp8_linear(input: torch.Tensor, data: torch.Tensor, scales: torch.Tensor) -> torch.Tensor:
    """``input @ W.T`` for weights kept in 8 bits: ``data``, ``scales = fp8_quantize(W, (128, 128))``.  ``input`` is [M, K] in float16 or
    bfloat16 (under autocast: cast to its dtype), quantized by the call in (1, 128) blocks; the result has its dtype.  Few rows (16, and up
    to 64 of small layers) run in one launch.  No gradient: the call is refused where one would be recorded."""
    return _loader.bridge().fp8_linear(input, data, scales)


@traceable
def blockwise_dropout_matmul_fp8_mask(input: torch.Tensor, mask: torch.Tensor, block_size, p: float,
                                      weight: torch.Tensor) -> torch.Tensor:
    """:func:`blockwise_dropout_matmul_fp8` with the mask given (True = dropped)."""
    if not 0 <= p < 1:
        raise ValueError("Dropout probability must be in [0, 1)")
    return _loader.bridge().linear_fp8(input, weight, mask, _block_size(block_size), p, None, None)


@traceable
def blockwise_dropout_matmul_fp8(input: torch.Tensor, weight: torch.Tensor, block_size, p: float,
                                 seed: int | None = None) -> torch.Tensor:
    """``(keep ⊙ input)/(1-p) @ weight.T`` and both gradients from operands in 8 bits, with a fresh block mask that is drawn as
    :func:`hip_blockwise_dropout_matmul` draws it (``seed`` pins it).  ``block_size``: a multiple of 128.

    For the backward the call keeps the input and the weight in 8 bits, each where its gradient is wanted, not the 16-bit tensors."""
    if not 0 <= p < 1:
        raise ValueError("Dropout probability must be in [0, 1)")
    return _loader.bridge().linear_fp8(input, weight, None, _block_size(block_size), p, *draw_source(input, seed))
