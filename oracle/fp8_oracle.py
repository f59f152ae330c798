"""Definitions in 64 bits of the 8-bit matrices, their products and the AdamW step, in numpy.

Nothing here shares code with the package: values are put on a format's grid by arithmetic, not by codes."""
from __future__ import annotations

import numpy as np

BLOCK = 128


def to_grid(y: np.ndarray, least: float, dither=None) -> np.ndarray:
    """Magnitudes on the grid of three bits of mantissa, normal from ``least`` on: nearest (halves to even), or down after
    ``dither`` of a grid step was added."""
    _, e = np.frexp(np.maximum(y, least))
    grid = np.ldexp(1.0, e - 4)
    steps = np.rint(y / grid) if dither is None else np.floor(y / grid + dither)
    return steps * grid


def least_power(most: np.ndarray, limit: float) -> np.ndarray:
    """The least power of two (2^-127 .. 2^127) that times ``limit`` reaches ``most``; 1 for zero."""
    _, e = np.frexp(most / limit)
    p = np.ldexp(1.0, e)
    p = np.where(most <= limit * p / 2, p / 2, p)  # (an exact power: frexp's mantissa is a half)
    return np.where(most > 0, np.clip(p, 2.0 ** -127, 2.0 ** 127), 1.0)


def quantize(x: np.ndarray, side: int):
    """(values, scales) of a matrix in e4m3 with a power of two for each ``side`` x 128 block; NaN for what is not finite."""
    x = np.asarray(x, dtype=np.float64)
    r, c = x.shape
    rb, cb = -(-r // side), -(-c // BLOCK)
    wide = np.zeros((rb * side, cb * BLOCK))
    wide[:r, :c] = x
    finite = np.where(np.isfinite(wide), np.abs(wide), 0.0)
    scales = least_power(finite.reshape(rb, side, cb, BLOCK).max(axis=(1, 3)), 448.0)
    by = np.repeat(np.repeat(scales, side, 0), BLOCK, 1)
    values = np.where(np.isfinite(wide), np.copysign(to_grid(finite / by, 2.0 ** -6), wide) * by, np.nan)
    return values[:r, :c], scales


def magnitudes(x: np.ndarray, side: int) -> np.ndarray:
    """What the matrix cores take an element's size for, over whole 128-blocks: at least that of the least normal code, 2^-6 of
    its scale, since the exponent of smaller codes and of zero is the same."""
    values, scales = quantize(x, side)
    r, c = values.shape
    least = np.repeat(np.repeat(scales, side, 0), BLOCK, 1)[:r] * 2.0 ** -6
    wide = np.zeros_like(least)
    wide[:, :c] = np.abs(values)
    return np.maximum(wide, least)


def product(a: np.ndarray, a_side: int, b: np.ndarray, b_side: int):
    """(A B^T, the sums of its terms' sizes) of two matrices in 8 bits."""
    return quantize(a, a_side)[0] @ quantize(b, b_side)[0].T, magnitudes(a, a_side) @ magnitudes(b, b_side).T


def keep_matrix(mask: np.ndarray, bs: int, rows: int, cols: int) -> np.ndarray:
    return (~np.repeat(np.repeat(mask, bs, 0), bs, 1))[:rows, :cols].astype(np.float64)


def train(x, w, dy, mask, bs: int, p: float):
    """(Y, dX, dW) of the block-dropout linear layer in 8 bits, and the sums of their terms' sizes."""
    s = 1.0 / (1.0 - p)
    keep = keep_matrix(mask, bs, *x.shape)
    # (a dropped block isn't read: what is not finite in it stays out)
    x = np.where(keep > 0, x, 0.0)
    y, sy = product(x, 1, w, BLOCK)
    dx, sdx = product(dy, 1, w.T, BLOCK)
    dw, sdw = product(dy.T, 1, x.T, 1)
    return (s * y, s * dx * keep, s * dw), (s * sy, s * sdx * keep, s * sdw)


# ---- AdamW ------------------------------------------------------------------------------------------------------------------
FORMATS = {"first": (448.0, 2.0 ** -6, 7), "second": (61440.0, 2.0 ** -14, 15)}


def dither(n: int, step: int, which: str) -> np.ndarray:
    """The random bits of a step, over 2^16: O'Neill's 32-bit RXS-M-XS generator one step behind element + step * 0x9E3779B1."""
    word = np.uint64(0xFFFFFFFF)
    s = (np.arange(n, dtype=np.uint64) + np.uint64(step * 0x9E3779B1 & 0xFFFFFFFF)) & word
    s = (s * np.uint64(747796405) + np.uint64(2891336453)) & word
    s = (((s >> ((s >> np.uint64(28)) + np.uint64(4))) ^ s) * np.uint64(277803737)) & word
    s = (s >> np.uint64(22)) ^ s
    bits = s >> np.uint64(16) if which == "first" else s & np.uint64(0xFFFF)
    return bits.astype(np.float64) / 65536.0


def rounded_state(x: np.ndarray, which: str, step: int) -> np.ndarray:
    """The values of an average after it was put into 8 bits at ``step``."""
    limit, least, _ = FORMATS[which]
    n = x.size
    wide = np.zeros(-(-n // BLOCK) * BLOCK)
    wide[:n] = np.abs(x.reshape(-1))
    scales = least_power(wide.reshape(-1, BLOCK).max(1), limit)
    y = wide / np.repeat(scales, BLOCK)
    y = to_grid(y[:n], least, dither(n, step, which)) * np.repeat(scales, BLOCK)[:n]
    return np.copysign(y, x.reshape(-1)).reshape(x.shape)


def state_table(which: str) -> np.ndarray:
    """The values of the 256 codes (those of e4m3's NaNs and of the second format's largest exponent aside)."""
    _, _, bias = FORMATS[which]
    bits = 4 if which == "first" else 5
    half = [j * 2.0 ** (1 - bias - 3) if i == 0 else (8 + j) * 2.0 ** (i - bias - 3) for i in range(1 << bits) for j in range(8)]
    table = np.array(half + [-v for v in half] if which == "first" else half)
    if which == "first":
        table[[127, 255]] = np.nan
    else:
        table[248], table[249:] = np.inf, np.nan
    return table


def adamw(p, g, m, v, step: int, lr, beta1, beta2, eps, decay):
    """(p, m, v) after step number ``step``, the averages not yet rounded."""
    p, g, m, v = (np.asarray(t, dtype=np.float64) for t in (p, g, m, v))
    m = beta1 * m + (1.0 - beta1) * g
    v = beta2 * v + (1.0 - beta2) * g * g
    p = p * (1.0 - lr * decay) - lr * (m / (1.0 - beta1 ** step)) / (np.sqrt(v / (1.0 - beta2 ** step)) + eps)
    return p, m, v
