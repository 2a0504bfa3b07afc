"""CPU oracle for the attention over packed sequences — TEST INFRASTRUCTURE ONLY.

Nothing in the product path imports this module. NumPy, float64 from the given inputs:

* ``attention`` / ``attention_vjp``: per sequence and head, the softmax over the seen keys and its transpose,
  written row by row from the definition; queries that see no key give zeros, rows outside every sequence
  are zeros.
* ``bounds``: how far a computation with weights and outputs rounded by at most ``u`` relative (half a step of
  the type) and sums in f32 may be off, element by element. With f = (terms + 16) 2^-24 for the sums and
  e_p for a softmax weight (twice the error of its score, and the sum's):
      out   A (u + e_p + f) + u |out|,                A = sum p |v|
      delta sum |do| (out's + f |out|)
      ds    p (f sum |do| |v| + delta's) + |ds| (u + e_p + f)
      dq    scale sum (ds's + f |ds|) |k| + u |dq|, and dk alike; dv  sum p (u + e_p + f) |do| + u |dv|.
  f32 ends at 2^-126: the exponential and the matrix units give 0 for less. So a weight, a score gradient
  and a product are each off by up to 2^-126 more than relative errors say. A term of a sum has a weight or a
  gradient p (dp - delta), which is off by up to 2^-126 (1 + |dp - delta|), times a row's element, and is a
  product itself: 2^-126 (1 + (1 + |dp - delta|) |element|) a term, taken with the largest of each.
"""

from __future__ import annotations

import numpy as np

__all__ = ["attention", "attention_vjp", "bounds", "sequences"]


def sequences(offsets, key_offsets=None, key_lengths=None):
    """``(q0, n, k0, m)`` of each sequence."""
    key_offsets = offsets if key_offsets is None else key_offsets
    out = []
    for i in range(len(offsets) - 1):
        m = key_offsets[i + 1] - key_offsets[i] if key_lengths is None else key_lengths[i]
        out.append((int(offsets[i]), int(offsets[i + 1] - offsets[i]), int(key_offsets[i]), int(m)))
    return out


def _weights(q, k, scale, causal):
    """Softmax weights ``[n, m]`` of one head; unseen pairs and rows without keys weigh 0."""
    n, m = q.shape[0], k.shape[0]
    s = (q @ k.T) * scale
    seen = np.ones((n, m), bool)
    if causal:
        seen = np.arange(m)[None, :] <= np.arange(n)[:, None] + (m - n)
    p = np.zeros((n, m))
    for t in range(n):
        if seen[t].any():
            e = np.exp(s[t, seen[t]] - s[t, seen[t]].max())
            p[t, seen[t]] = e / e.sum()
    return p, s, seen


def _heads(q, k, v, seqs, *more):
    """Views of every (sequence, head): rows of q (and of `more`), rows of k and v."""
    group = q.shape[1] // k.shape[1]
    for q0, n, k0, m in seqs:
        if n and m:
            for h in range(q.shape[1]):
                a, b = (slice(q0, q0 + n), h), (slice(k0, k0 + m), h // group)
                yield a, b, q[a], k[b], v[b], *(x[a] for x in more)


def attention(q, k, v, seqs, causal=True, scale=None):
    """``[T, H, D]`` float64."""
    q, k, v = (np.asarray(x, np.float64) for x in (q, k, v))
    scale = q.shape[2] ** -0.5 if scale is None else scale
    out = np.zeros(q.shape)
    for a, _, qh, kh, vh in _heads(q, k, v, seqs):
        out[a] = _weights(qh, kh, scale, causal)[0] @ vh
    return out


def attention_vjp(q, k, v, grad, seqs, causal=True, scale=None):
    """``(dq, dk, dv)`` for the cotangent ``grad``."""
    q, k, v, grad = (np.asarray(x, np.float64) for x in (q, k, v, grad))
    scale = q.shape[2] ** -0.5 if scale is None else scale
    dq, dk, dv = (np.zeros(x.shape) for x in (q, k, v))
    for a, b, qh, kh, vh, g in _heads(q, k, v, seqs, grad):
        p = _weights(qh, kh, scale, causal)[0]
        dv[b] += p.T @ g
        dp = g @ vh.T
        ds = p * (dp - (p * dp).sum(-1, keepdims=True)) * scale
        dq[a] = ds @ kh
        dk[b] += ds.T @ qh
    return dq, dk, dv


def bounds(q, k, v, grad, seqs, u, causal=True, scale=None):
    """The largest errors of ``(out, dq, dk, dv)``, element by element."""
    q, k, v, grad = (np.asarray(x, np.float64) for x in (q, k, v, grad))
    d = q.shape[2]
    scale = d ** -0.5 if scale is None else scale
    eps = 2.0 ** -24
    out, dq, dk, dv = (np.zeros(x.shape) for x in (q, q, k, v))
    sums = [np.zeros(x.shape) for x in (k, v)]
    tiny = 2.0 ** -126
    for a, b, qh, kh, vh, g in _heads(q, k, v, seqs, grad):
        n, m = qh.shape[0], kh.shape[0]
        p, s, seen = _weights(qh, kh, scale, causal)
        f, fq = (m + d + 16) * eps, (n * q.shape[1] // k.shape[1] + d + 16) * eps
        # a score's products and sum, its scaling and the reference score taken off it
        es = scale * (d + 2) * eps * (np.abs(qh) @ np.abs(kh).T) + 4 * eps * np.abs(s)
        ep = 2 * np.where(seen, es, 0.0).max(-1, keepdims=True) + (m + 16) * eps
        o, reach = p @ vh, p @ np.abs(vh)
        out[a] = reach * (u + ep + f) + u * np.abs(o)
        dp = g @ vh.T
        delta = (g * o).sum(-1, keepdims=True)
        e_delta = (np.abs(g) * (out[a] + f * np.abs(o))).sum(-1, keepdims=True)
        ds = p * (dp - delta)
        e_ds = p * ((d + 16) * eps * (np.abs(g) @ np.abs(vh).T) + e_delta) + np.abs(ds) * (u + ep + f)
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
