"""CPU oracle for packed attention with shaped scores — TEST INFRASTRUCTURE ONLY.

Nothing in the product path imports this module. NumPy, float64 from the given inputs. With place = t + m - n:

    x = cap tanh(scale q.k / cap) - slope_h |place - j|     (without a cap: scale q.k - ...)
    seen: |place - j| < window and (not causal or j <= place or j < prefix)

* ``attention`` / ``attention_vjp``: per sequence and head, the softmax over the seen keys and its transpose; queries
  that see no key give zeros, rows outside every sequence are zeros.
* ``bounds``: how far a computation with weights, their gradients and outputs rounded by at most ``u`` relative (half a
  step of the type) and everything else in f32 may be off, element by element. As in packed_attention_ref, with
      e_t   of tanh:   ``bend`` |t| + 8 2^-24 + (error of scale q.k) / cap
      e_x   of x:      cap e_t (or that of scale q.k) + 2^-24 (4 |x| + 4 slope |place - j| + 4 |log sum exp|)
      e_p   of a weight, relative: its e_x and the row's mean of them, and the sum's
      e_c   of 1 - t^2: 2 |t| e_t + 4 2^-24, and a gradient ds (1 - t^2) is off by e_ds (1 - t^2) + |ds| e_c.
  ``bend`` is the relative error of the tanh's polynomial: 7.3e-7 beside bf16 tensors, 1e-7 beside f32.
"""

from __future__ import annotations

import numpy as np

__all__ = ["attention", "attention_vjp", "bounds", "Shape"]


class Shape:
    def __init__(self, causal=True, scale=None, cap=None, slopes=None, window=None, prefixes=None):
        self.causal, self.scale, self.cap, self.slopes, self.window, self.prefixes = causal, scale, cap, slopes, window, prefixes

    def scores(self, q, k, head, seq):
        """(raw scores, tanh, x, distance, seen) of one head of one sequence."""
        n, m = q.shape[0], k.shape[0]
        place, key = np.arange(n)[:, None] + (m - n), np.arange(m)[None, :]
        distance = np.abs(place - key)
        seen = np.ones((n, m), bool)
        if self.causal:
            prefix = 0 if self.prefixes is None else self.prefixes[seq]
            seen = (key <= place) | (key < prefix)
        if self.window is not None:
            seen = seen & (distance < self.window)
        s = (q @ k.T) * (q.shape[1] ** -0.5 if self.scale is None else self.scale)
        t = np.zeros_like(s) if self.cap is None else np.tanh(s / self.cap)
        x = s if self.cap is None else self.cap * t
        slope = 0.0 if self.slopes is None else float(self.slopes[head])
        return s, t, x - slope * distance, slope * distance, seen


def _softmax(x, seen):
    p, lse = np.zeros(x.shape), np.zeros((x.shape[0], 1))
    for r in range(x.shape[0]):
        if seen[r].any():
            top = x[r, seen[r]].max()
            e = np.exp(x[r, seen[r]] - top)
            p[r, seen[r]] = e / e.sum()
            lse[r] = top + np.log(e.sum())
    return p, lse


def _heads(q, k, seqs):
    group = q.shape[1] // k.shape[1]
    for i, (q0, n, k0, m) in enumerate(seqs):
        if n and m:
            for h in range(q.shape[1]):
                yield i, h, (slice(q0, q0 + n), h), (slice(k0, k0 + m), h // group)


def attention(q, k, v, seqs, shape):
    q, k, v = (np.asarray(x, np.float64) for x in (q, k, v))
    out = np.zeros(q.shape)
    for i, h, a, b in _heads(q, k, seqs):
        _, _, x, _, seen = shape.scores(q[a], k[b], h, i)
        out[a] = _softmax(x, seen)[0] @ v[b]
    return out


def attention_vjp(q, k, v, grad, seqs, shape):
    q, k, v, grad = (np.asarray(x, np.float64) for x in (q, k, v, grad))
    scale = q.shape[2] ** -0.5 if shape.scale is None else shape.scale
    dq, dk, dv = (np.zeros(x.shape) for x in (q, k, v))
    for i, h, a, b in _heads(q, k, seqs):
        _, t, x, _, seen = shape.scores(q[a], k[b], h, i)
        p = _softmax(x, seen)[0]
        dp = grad[a] @ v[b].T
        ds = p * (dp - (p * dp).sum(-1, keepdims=True)) * (1 - t * t) * scale
        dv[b] += p.T @ grad[a]
        dq[a] = ds @ k[b]
        dk[b] += ds.T @ q[a]
    return dq, dk, dv


def bounds(q, k, v, grad, seqs, u, shape):
    """The largest errors of ``(out, dq, dk, dv)``, element by element."""
    q, k, v, grad = (np.asarray(x, np.float64) for x in (q, k, v, grad))
    d, eps, tiny = q.shape[2], 2.0 ** -24, 2.0 ** -126
    bend = 7.3e-7 if u > 2.0 ** -20 else 1e-7
    scale = d ** -0.5 if shape.scale is None else shape.scale
    out, dq, dk, dv = (np.zeros(x.shape) for x in (q, q, k, v))
    sums = [np.zeros(x.shape) for x in (k, v)]
    for i, h, a, b in _heads(q, k, seqs):
        qh, kh, vh, g = q[a], k[b], v[b], grad[a]
        n, m = qh.shape[0], kh.shape[0]
        s, t, x, away, seen = shape.scores(qh, kh, h, i)
        p, lse = _softmax(x, seen)
        f, fq = (m + d + 16) * eps, (n * q.shape[1] // k.shape[1] + d + 16) * eps
        es = scale * (d + 2) * eps * (np.abs(qh) @ np.abs(kh).T) + 4 * eps * np.abs(s)
        et = np.zeros_like(s) if shape.cap is None else bend * np.abs(t) + 8 * eps + es / shape.cap
        ex = (es if shape.cap is None else shape.cap * et) + 4 * eps * (np.abs(x) + away + np.abs(lse))
        ep = ex + (p * ex).sum(-1, keepdims=True) + (m + 16) * eps
        c, ec = 1 - t * t, np.zeros_like(s) if shape.cap is None else 2 * np.abs(t) * et + 4 * eps
        o = p @ vh
        out[a] = (p * (u + ep + f)) @ np.abs(vh) + u * np.abs(o)
        dp = g @ vh.T
        delta = (g * o).sum(-1, keepdims=True)
        e_delta = (np.abs(g) * (out[a] + f * np.abs(o))).sum(-1, keepdims=True)
        ds = p * (dp - delta)
        e_ds = (p * ((d + 16) * eps * (np.abs(g) @ np.abs(vh).T) + e_delta) + np.abs(ds) * (u + ep + f)) * c + np.abs(ds) * ec
        ds = ds * c
        dq[a] = scale * (e_ds + f * np.abs(ds)) @ np.abs(kh) + u * scale * np.abs(ds @ kh)
        dk[b] += scale * (e_ds + fq * np.abs(ds)).T @ np.abs(qh)
        dv[b] += (p * (u + ep + fq)).T @ np.abs(g)
        most = 1 + np.abs(dp - delta).max()
        out[a] += m * tiny * (1 + np.abs(vh).max())
        dq[a] += m * tiny * (1 + most * np.abs(kh).max()) * max(scale, 1)
        dk[b] += n * tiny * (1 + most * np.abs(qh).max()) * max(scale, 1)
        dv[b] += n * tiny * (1 + np.abs(g).max())
        sums[0][b] += scale * ds.T @ qh
        sums[1][b] += p.T @ g
    return out, dq, dk + u * np.abs(sums[0]), dv + u * np.abs(sums[1])
