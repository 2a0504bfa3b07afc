"""CPU oracle for the rotary positions on several axes — TEST INFRASTRUCTURE ONLY.

``rotate``: every pair of channels as a complex number times ``exp(i angle)``, float64 (``sign = -1``: the
gradient). ``angles``: ``position * base ** -e`` in float64 (int64 positions below 2^53 are exact).
"""

from __future__ import annotations

import numpy as np

__all__ = ["angles", "rotate"]


def angles(positions, sections, base=10000.0, shared=False):
    """``[..., n]`` angles of positions ``[..., A]``."""
    positions = np.asarray(positions).astype(np.float64)
    n, columns = sum(sections), []
    for a, count in enumerate(sections):
        for j in range(count):
            e = len(columns) / n if shared else j / count
            columns.append(positions[..., a] * float(base) ** -e)
    return np.stack(columns, -1)


def rotate(x, positions, sections, base=10000.0, shared=False, interleaved=False, sign=1.0):
    """``[..., H, D]`` float64."""
    x = np.asarray(x, np.float64)
    n = sum(sections)
    a = angles(positions, sections, base, shared)[..., None, :]
    first, second = (slice(0, 2 * n, 2), slice(1, 2 * n, 2)) if interleaved else (slice(0, n), slice(n, 2 * n))
    z = (x[..., first] + 1j * x[..., second]) * np.exp(1j * sign * a)
    out = x.copy()
    out[..., first], out[..., second] = z.real, z.imag
    return out
