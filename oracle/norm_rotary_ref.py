"""CPU oracle for the norms with rotary positions — TEST INFRASTRUCTURE ONLY.

Nothing in the product path imports this module. NumPy, float64 from the given inputs:

* ``forward``: y = R (x r w), r = (mean x^2 + eps)^-1/2, the rotation by rotary_ref.
* ``backward``: g = R^T dy, dw = sum g x r, dx = r (g w - x r^2 mean(g w x)).
* ``forward_bound`` / ``backward_bounds``: how far a computation in f32, rounded once by at most ``u`` relative, may be off,
  element by element. With e = 2^-24: r is off by (D + 4) e of itself (the sum's terms are all of one sign; half of its
  relative error, the division, the root), a normed channel by (D + 8) e, cos and sin by 4 e absolute (their own
  rounding, that of the reduced angle, at most 2^-25 turns: 2 pi 2^-25 < 4 e), a product of the rotation by 2 e:
      y      sum over the pair of |x r w| times (D + 16) e, and u |y|
      g      e_g = 8 e (|dy_a| + |dy_b|)
      u x    e_m = mean((|g w x|) (D + 8) e + e_g |w x|)
      dx     r (e_g |w| + |x| r^2 e_m) + (2 D + 32) e (r |g w| + r^3 |x| mean|g w x|) + u |dx|
      dw     sum (e_g |x r| + (D + 16 + min(rows, 4096)) e |g x r|) + u_w |dw|
  and 2^-126 more for each of two products, which f32 does not hold below.
"""

from __future__ import annotations

import numpy as np

from . import rotary_ref

__all__ = ["forward", "backward", "forward_bound", "backward_bounds"]

E, TINY = 2.0 ** -24, 2.0 ** -125


def _turn(x, positions, sections, kw, sign=1.0):
    return rotary_ref.rotate(x, positions, sections, sign=sign, **kw)


def _pair_sum(x, sections, interleaved):
    """|x| of both channels of each pair, for each of them; channels behind the pairs as they are."""
    x, n = np.abs(x), sum(sections)
    out = x.copy()
    a, b = (slice(0, 2 * n, 2), slice(1, 2 * n, 2)) if interleaved else (slice(0, n), slice(n, 2 * n))
    out[..., a] = out[..., b] = x[..., a] + x[..., b]
    return out


def _root(x, eps):
    return 1.0 / np.sqrt((x * x).mean(-1, keepdims=True) + eps)


def forward(x, w, positions, sections, eps, **kw):
    x = np.asarray(x, np.float64)
    w = 1.0 if w is None else np.asarray(w, np.float64)
    return _turn(x * _root(x, eps) * w, positions, sections, kw)


def backward(x, w, dy, positions, sections, eps, **kw):
    """(dx, dw); dw also without a weight, whose gradient it then is at ones."""
    x, dy = np.asarray(x, np.float64), np.asarray(dy, np.float64)
    w = np.ones(x.shape[-1]) if w is None else np.asarray(w, np.float64)
    r, g = _root(x, eps), _turn(dy, positions, sections, kw, -1.0)
    u = g * w
    return r * (u - x * r * r * (u * x).mean(-1, keepdims=True)), (g * x * r).sum((0, 1))


def forward_bound(x, w, positions, sections, eps, u, **kw):
    x = np.asarray(x, np.float64)
    w = 1.0 if w is None else np.asarray(w, np.float64)
    n = x * _root(x, eps) * w
    y = _turn(n, positions, sections, kw)
    e = _pair_sum(n, sections, kw.get("interleaved", False)) * (x.shape[-1] + 16) * E
    return e + u * (np.abs(y) + e) + TINY


def backward_bounds(x, w, dy, positions, sections, eps, u, u_w, **kw):
    x, dy = np.asarray(x, np.float64), np.asarray(dy, np.float64)
    w = np.ones(x.shape[-1]) if w is None else np.asarray(w, np.float64)
    d, rows = x.shape[-1], x.shape[0] * x.shape[1]
    r, g = _root(x, eps), _turn(dy, positions, sections, kw, -1.0)
    e_g = 8 * E * _pair_sum(dy, sections, kw.get("interleaved", False)) + TINY
    gwx = np.abs(g * w * x)
    e_m = (gwx * (d + 8) * E + e_g * np.abs(w * x) + TINY).mean(-1, keepdims=True)
    dx, dw = backward(x, w, dy, positions, sections, eps, **kw)
    e = r * (e_g * np.abs(w) + np.abs(x) * r * r * e_m) + (2 * d + 32) * E * (r * np.abs(g * w) + r ** 3 * np.abs(x) * gwx.mean(-1, keepdims=True)) + TINY * (1 + r)
    e_w = (e_g * np.abs(x * r) + (d + 16 + min(rows, 4096)) * E * np.abs(g * x * r) + TINY).sum((0, 1))
    return e + u * (np.abs(dx) + e), e_w + u_w * (np.abs(dw) + e_w)
