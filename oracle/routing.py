"""Routing to experts in float64, one token after the other: choice, gradient, sort, weighted sum.

The reference has no routing; these follow the definitions of the entry points in include/mi355x_bench.h.
"""

from __future__ import annotations

import numpy as np


def scores(logits, kind):
    """Softmax or sigmoid of one token's logits; a masked (-inf) logit scores 0, a row of them all 0."""
    logits = np.asarray(logits, dtype=np.float64)
    if kind == "sigmoid":
        with np.errstate(over="ignore"):
            return 1 / (1 + np.exp(-logits))
    largest = logits.max()
    if largest == -np.inf:
        return np.zeros_like(logits)
    with np.errstate(invalid="ignore"):
        powers = np.exp(logits - largest)
    return powers / powers.sum()


def _ranked(values, indices):
    """Indices by falling value, of equal ones the lower first; values of -inf left out."""
    return sorted((i for i in indices if values[i] > -np.inf), key=lambda i: (-values[i], i))


def route(logits, top, bias=None, kind="softmax", groups=1, top_groups=1, renormalize=True, scale=1.0):
    """(experts, weights) [tokens][top]."""
    logits = np.asarray(logits, dtype=np.float64)
    tokens, count = logits.shape
    experts = np.full((tokens, top), -1, dtype=np.int32)
    weights = np.zeros((tokens, top))
    size = count // groups
    for t in range(tokens):
        s = scores(logits[t], kind)
        c = s if bias is None else s + np.asarray(bias, dtype=np.float64)
        c = np.where(np.isnan(c), -1e38, c)
        c = np.where(logits[t] == -np.inf, -np.inf, c)
        kept = range(count)
        if groups > 1:
            group = []
            for g in range(groups):
                best = sorted((v for v in c[g * size:(g + 1) * size] if v > -np.inf), reverse=True)[:2]
                group.append(sum(best) if best else -np.inf)
            order = sorted(range(groups), key=lambda g: (-group[g], g))[:top_groups]
            kept = [i for i in range(count) if i // size in order]
        chosen = _ranked(c, kept)[:top]
        experts[t, :len(chosen)] = chosen
        w = s[chosen]
        if renormalize and len(chosen):
            total = w.sum()
            w = np.zeros_like(w) if total == 0 else w / total
        weights[t, :len(chosen)] = w * scale
    return experts, weights


def route_backward(logits, experts, d_weights, kind="softmax", renormalize=True, scale=1.0):
    """d_logits by the chain of the weights' Jacobian: w = scale * s_j / sum s, s = softmax or sigmoid."""
    logits = np.asarray(logits, dtype=np.float64)
    d_logits = np.zeros_like(logits)
    for t in range(logits.shape[0]):
        s = scores(logits[t], kind)
        entries = [j for j in range(experts.shape[1]) if experts[t, j] >= 0]
        chosen = [int(experts[t, j]) for j in entries]
        g = np.array([d_weights[t, j] for j in entries]) * scale
        if renormalize and chosen:
            total = s[chosen].sum()
            jacobian = (np.eye(len(chosen)) - (s[chosen] / total)[:, None]) / total if total else np.zeros((len(chosen),) * 2)
            g = g @ jacobian  # d w_i / d s_j = (delta_ij - s_i / sum) / sum
        d_scores = np.zeros_like(s)
        d_scores[chosen] = g
        if kind == "sigmoid":
            d_logits[t] = d_scores * s * (1 - s)
        else:
            d_logits[t] = s * (d_scores - d_scores @ s)
    return d_logits


def dispatch(experts, count):
    """(offsets, order, slots)."""
    flat = np.asarray(experts).reshape(-1)
    members = [[i for i, e in enumerate(flat) if e == x] for x in range(count)]
    order = np.array([i for m in members for i in m] + [-1] * sum(1 for e in flat if not 0 <= e < count), dtype=np.int64)
    offsets = np.concatenate([[0], np.cumsum([len(m) for m in members])])
    slots = np.full(flat.shape, -1, dtype=np.int64)
    for slot, i in enumerate(order):
        if i >= 0:
            slots[i] = slot
    return offsets, order, slots.reshape(np.asarray(experts).shape)


def combine(y, slots, weights):
    """(out, the same sum of magnitudes)."""
    y, weights = np.asarray(y, dtype=np.float64), np.asarray(weights, dtype=np.float64)
    out, size = np.zeros((slots.shape[0], y.shape[1])), np.zeros((slots.shape[0], y.shape[1]))
    for t, row in enumerate(slots):
        for j, slot in enumerate(row):
            if 0 <= slot < y.shape[0]:
                out[t] += weights[t, j] * y[slot]
                size[t] += np.abs(weights[t, j] * y[slot])
    return out, size


def combine_backward(d_out, y, slots, weights):
    """(d_y, d_weights, the magnitudes of d_weights' sums); rows of d_y that no slot names are zero."""
    d_out, y = np.asarray(d_out, dtype=np.float64), np.asarray(y, dtype=np.float64)
    d_y, d_weights = np.zeros_like(y), np.zeros(slots.shape)
    size = np.zeros(slots.shape)
    for t, row in enumerate(slots):
        for j, slot in enumerate(row):
            if 0 <= slot < y.shape[0]:
                d_y[slot] = weights[t, j] * d_out[t]
                d_weights[t, j] = d_out[t] @ y[slot]
                size[t, j] = np.abs(d_out[t]) @ np.abs(y[slot])
    return d_y, d_weights, size
