"""Root-mean-square norm of rows and its gradients in float64. The reference has none."""

from __future__ import annotations

import numpy as np


def _inverse(total, eps):
    return 1.0 / np.sqrt((total * total).mean(axis=1, keepdims=True) + eps)


def rms_norm(total, weight, eps):
    """total * weight / sqrt(mean(total^2) + eps)."""
    total = np.asarray(total, dtype=np.float64)
    return total * _inverse(total, eps) * weight


def rms_norm_backward(d_out, total, weight, eps, d_total=None):
    """(d_x, d_weight)."""
    total = np.asarray(total, dtype=np.float64)
    inverse = _inverse(total, eps)
    d_normed = d_out * weight
    along = (d_normed * total).mean(axis=1, keepdims=True)
    d_x = inverse * d_normed - total * inverse**3 * along
    return d_x if d_total is None else d_x + d_total, (d_out * total * inverse).sum(axis=0)
