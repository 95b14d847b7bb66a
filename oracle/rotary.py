"""Oracle of the rotary positions with several axes, in float64: pairs of channels as complex
numbers, turned by exp(i theta)."""

from __future__ import annotations

import numpy as np


def rotary(x, positions, inv_freq, sections, interleaved=False, inverse=False):
    """``x [T, H, D]``, ``positions [T, axes]``; frequency i belongs to the axis of its section."""
    x = np.asarray(x, np.float64)
    axis = np.repeat(np.arange(len(sections)), sections)
    theta = np.asarray(positions, np.float64)[:, axis] * np.asarray(inv_freq, np.float64)
    turn = np.exp((-1j if inverse else 1j) * theta)[:, None]
    half = len(axis)
    i = np.arange(half)
    first, second = (2 * i, 2 * i + 1) if interleaved else (i, i + half)
    z = (x[..., first] + 1j * x[..., second]) * turn
    y = x.copy()
    y[..., first], y[..., second] = z.real, z.imag
    return y
