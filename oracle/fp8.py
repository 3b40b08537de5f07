"""FP8 operands with block scales in float64: the format, its quantisation, the products and the gated pair.

The reference has none of these; the rules are this library's (the largest magnitude of a block decides the smallest
power of two that keeps it within E4M3's 448), on the OCP 8-bit format E4M3 and its scale format E8M0.
"""

from __future__ import annotations

import numpy as np

BLOCK, STEP = 128, 512


def _grid():
    """Magnitudes of E4M3's codes 0 .. 126, in their order."""
    code = np.arange(127)
    field, fraction = code >> 3, code & 7
    return np.where(field == 0, fraction * 2.0**-9, (8 + fraction) * 2.0**(field - 10.0))


GRID = _grid()


def _largest(x, block):
    """Largest magnitudes [ceil(rows/block)][ceil(k/128)], and whether a block is finite."""
    rows, k = x.shape
    padded = np.pad(x, ((0, -rows % block), (0, -k % BLOCK)))
    blocks = padded.reshape(padded.shape[0] // block, block, padded.shape[1] // BLOCK, BLOCK)
    finite = np.isfinite(blocks).all(axis=(1, 3))
    return np.abs(np.where(np.isfinite(blocks), blocks, 0.0)).max(axis=(1, 3), initial=0.0), finite


def scale_codes(x, block=1):
    """E8M0 codes [ceil(rows/block)][ceil(k/128)] of float64 rows x."""
    largest, finite = _largest(x, block)
    fraction, power = np.frexp(np.where(largest > 0, largest, 1.0))  # largest = f * 2^power, f in [0.5, 1)
    exponent = power - 9 + (fraction > 0.875)
    exponent = np.where(largest > 0, np.maximum(exponent, -127), -127)
    return np.where(finite, exponent + 127, 255).astype(np.uint8)


def _spread(scales, rows, k, block):
    return np.repeat(np.repeat(scales, block, axis=0)[:rows], BLOCK, axis=1)[:, :k]


def element_codes(x, scales, block=1):
    """E4M3 codes [rows][k] of x under the scales: nearest, ties to the even code."""
    spread = _spread(scales, *x.shape, block)
    nan = spread == 255
    size = np.abs(np.where(nan, 0.0, x)) * np.exp2(127.0 - spread.astype(np.float64))
    upper = np.clip(np.searchsorted(GRID, size), 1, 126)
    below, above = size - GRID[upper - 1], GRID[upper] - size
    code = np.where((below < above) | ((below == above) & (upper % 2 == 1)), upper - 1, upper)
    return (code | np.where(np.signbit(x) & ~nan, 128, 0)).astype(np.uint8)


def quantize(x, block=1):
    """(codes [rows][k rounded up to 16], scales [ceil(k/512)][ceil(rows/block)][4]) of rows x."""
    x = np.asarray(x, dtype=np.float64)
    rows, k = x.shape
    scales = scale_codes(x, block)
    codes = np.pad(element_codes(x, scales, block), ((0, 0), (0, -k % 16)))
    steps = -(-k // STEP)
    padded = np.full((scales.shape[0], steps * 4), 127, dtype=np.uint8)
    padded[:, :scales.shape[1]] = scales
    return codes, padded.reshape(-1, steps, 4).transpose(1, 0, 2)


def values(codes, scales, k, block=1):
    """Float64 values [rows][k] of an operand; NaN where the scale is 255."""
    codes = codes[:, :k]
    flat = scales.transpose(1, 0, 2).reshape(scales.shape[1], -1)
    spread = _spread(flat, codes.shape[0], k, block)
    size = GRID[np.minimum(codes & 127, 126)] * np.exp2(spread.astype(np.float64) - 127)
    return np.where((spread == 255) | (codes & 127 == 127), np.nan, np.where(codes & 128, -size, size))


def rounded(x, block=1):
    """x as its operand holds it."""
    return values(*quantize(x, block), np.asarray(x).shape[1], block)


def linear(x, w):
    """Q(x) . Q(w)^T with w in blocks of 128 rows, and the same of the magnitudes (the scale of the rounding bound)."""
    a, b = rounded(x), rounded(w, BLOCK)
    return a @ b.T, np.abs(a) @ np.abs(b).T


def linear_backward(d_out, x, w):
    """((d_x, its magnitudes), (d_weight, its magnitudes)) of the linear layer, straight through."""
    d_rows, weight = rounded(d_out), rounded(w, BLOCK)
    d_columns, x_columns = rounded(np.asarray(d_out).T), rounded(np.asarray(x).T).T
    return ((d_rows @ weight, np.abs(d_rows) @ np.abs(weight)),
            (d_columns @ x_columns, np.abs(d_columns) @ np.abs(x_columns)))


def sigmoid(g):
    power = np.exp(-np.abs(g))
    return np.where(g >= 0, 1.0, power) / (1.0 + power)


def gate(pair):
    """silu(gate) * up of [gate | up]."""
    g, u = np.split(np.asarray(pair, dtype=np.float64), 2, axis=1)
    return g * sigmoid(g) * u


def gate_backward(d_out, pair):
    """The gradient of [gate | up]."""
    g, u = np.split(np.asarray(pair, dtype=np.float64), 2, axis=1)
    s = sigmoid(g)
    return np.concatenate([d_out * u * s * (1 + g * sigmoid(-g)), d_out * g * s], axis=1)
