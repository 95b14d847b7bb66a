"""Oracle of the norm of every head with the rotary positions on the result, and of its gradients, in float64."""

from __future__ import annotations

import numpy as np

from . import rotary as R


def normed_rotary(x, weight, eps, positions, inv_freq, sections, interleaved=False, grad=None):
    """``x [T, H, D]``, ``weight [D]`` or None.  Returns ``(y, y_size)`` and, with ``grad``, ``(dx, dx_size, dw,
    dw_size)`` as well: the sizes are sums of the absolute values that went into each element, of which an
    implementation in float32 is off by its roundings' part."""
    x = np.asarray(x, np.float64)
    w = np.ones(x.shape[-1]) if weight is None else np.asarray(weight, np.float64)
    how = (positions, inv_freq, sections, interleaved)
    half = sum(sections)
    i = np.arange(half)
    first, second = (2 * i, 2 * i + 1) if interleaved else (i, i + half)

    def pair_size(v):
        s = np.abs(v)
        both = s[..., first] + s[..., second]
        s[..., first] = s[..., second] = both
        return s

    r = 1.0 / np.sqrt((x * x).mean(-1, keepdims=True) + eps)
    n = x * r * w
    y = R.rotary(n, *how)
    if grad is None:
        return y, pair_size(n)
    grad = np.asarray(grad, np.float64)
    h, h_size = R.rotary(grad, *how, True), pair_size(grad)
    dot = (w * h * x).mean(-1, keepdims=True)
    dot_size = (np.abs(w) * h_size * np.abs(x)).mean(-1, keepdims=True)
    dx = r * (w * h - x * r * r * dot)
    dx_size = r * (np.abs(w) * h_size + np.abs(x) * r * r * dot_size)
    return y, pair_size(n), dx, dx_size, (h * x * r).sum((0, 1)), (h_size * np.abs(x) * r).sum((0, 1))
