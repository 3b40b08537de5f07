"""MXFP4 operands in float64: the format, its quantisation and the linear layer's products.

The reference has no MX quantisation (its MX FP4 rows draw codes, bench_tensor.py:55-69); the rules are the OCP
Microscaling format's, with the scale of a group that has no finite largest magnitude, and of zeros, fixed here.
"""

from __future__ import annotations

import numpy as np

GROUP, STEP = 32, 256
MAGNITUDES = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])


def scale_codes(x):
    """E8M0 codes [rows][ceil(k/32)] of float64 rows x."""
    rows, k = x.shape
    groups = np.pad(x, ((0, 0), (0, -k % GROUP))).reshape(rows, -1, GROUP)
    largest = np.abs(groups).max(axis=2) if groups.size else np.zeros(groups.shape[:2])
    finite = np.isfinite(groups).all(axis=2)
    _, power = np.frexp(np.where(finite, largest, 1.0))  # largest = f * 2^power, f in [0.5, 1)
    exponent = np.where(largest == 0, -127, np.clip(power - 1 - 2, -127, 127))
    return np.where(finite, exponent + 127, 255).astype(np.uint8)


def element_codes(x, scales):
    """E2M1 codes [rows][ceil(k/32)*32] of x under the given scales: nearest, ties to even, saturating at 6."""
    rows, k = x.shape
    groups = np.pad(x, ((0, 0), (0, -k % GROUP))).reshape(rows, -1, GROUP)
    nan = scales[..., None] == 255
    size = np.abs(np.where(nan, 0.0, groups)) * np.exp2(127.0 - scales[..., None].astype(np.float64))
    code = np.zeros(groups.shape, dtype=np.uint8)
    for lower in range(7):
        middle = (MAGNITUDES[lower] + MAGNITUDES[lower + 1]) / 2
        code += ((size >= middle) if lower % 2 else (size > middle)).astype(np.uint8)
    code |= np.where(np.signbit(groups) & ~nan, 8, 0).astype(np.uint8)
    return code.reshape(rows, -1)


def quantize(x):
    """(codes [rows][ceil(k/32)*16] two a byte, scales [ceil(k/256)][rows][8]) of rows x."""
    x = np.asarray(x, dtype=np.float64)
    rows, k = x.shape
    scales = scale_codes(x)
    code = element_codes(x, scales)
    blocks = -(-k // STEP)
    padded = np.full((rows, blocks * 8), 127, dtype=np.uint8)
    padded[:, :scales.shape[1]] = scales
    return code[:, 0::2] | code[:, 1::2] << 4, padded.reshape(rows, blocks, 8).transpose(1, 0, 2)


def values(codes, scales, k):
    """Float64 values [rows][k] of an operand; NaN where the scale is 255."""
    rows = codes.shape[0]
    code = np.stack([codes & 15, codes >> 4], axis=2).reshape(rows, -1)[:, :k]
    signed = np.where(code & 8, -1.0, 1.0) * MAGNITUDES[code & 7]
    column = np.arange(k)
    scale = scales[column // STEP, :, column % STEP // GROUP].T
    return np.where(scale == 255, np.nan, signed * np.exp2(scale.astype(np.float64) - 127))


def rounded(x):
    """x as its operand holds it."""
    return values(*quantize(x), np.asarray(x).shape[1])


def linear(x, w):
    """Q(x) . Q(w)^T, and the same of the magnitudes (the scale of the rounding bound)."""
    a, b = rounded(x), rounded(w)
    return a @ b.T, np.abs(a) @ np.abs(b).T


def linear_backward(d_out, x, w):
    """((d_x, its magnitudes), (d_weight, its magnitudes)) of the linear layer, straight through."""
    d_rows, w_columns = rounded(d_out), rounded(np.asarray(w).T).T
    d_columns, x_columns = rounded(np.asarray(d_out).T), rounded(np.asarray(x).T).T
    return ((d_rows @ w_columns, np.abs(d_rows) @ np.abs(w_columns)),
            (d_columns @ x_columns, np.abs(d_columns) @ np.abs(x_columns)))
