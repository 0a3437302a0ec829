"""The norm with its rotation in numpy, 64 bits, from the definition."""
import numpy as np


def norm_rope(x, w, cos, sin, eps, order):
    """x (T, H, 128), w (128), cos / sin (T, 64) of each token, float64. Returns the rows
    and, per element, the size of the terms that the rotation adds up."""
    x = np.asarray(x, np.float64)
    y = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * w
    a, b = y[..., :64], y[..., 64:]
    c, s = cos[:, None], sin[:, None]
    rows = np.concatenate([a * c - b * s, b * c + a * s], -1)
    size = np.concatenate([np.abs(a * c) + np.abs(b * s), np.abs(b * c) + np.abs(a * s)], -1)
    if order == "sorted_pair":  # sorted pair j = pair 63 - j, its two elements side by side
        perm = np.array([d for j in range(64) for d in (63 - j, 127 - j)])
        rows, size = rows[..., perm], size[..., perm]
    return rows, size


def bound(rows, size):
    """How far a bf16 result may be off: half a step of bf16 (2^-8 relative, 2^-134 below
    its normal range), and fp32's share: the sum of 128 squares is off by at most 128 steps
    of 2^-24 (half of that in the root), reciprocal root, two products and the rotation by
    fewer than 16 more, each relative to the terms."""
    return np.abs(rows) * 2.0 ** -8 + size * (80 * 2.0 ** -24) + 2.0 ** -133
