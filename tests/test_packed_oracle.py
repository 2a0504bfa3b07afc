"""The CPU oracles of packed attention and rotary positions against independent statements of the same:
torch float64 attention and autograd of the composed operations, finite differences, rotation matrices,
closed forms, and planted mistakes that have to fail."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import packed_attention_ref as PA
from oracle import rotary_ref as RO


def _inputs(seed, t, s, h, hk, d):
    rng = np.random.default_rng(seed)
    return [rng.standard_normal(x) for x in ((t, h, d), (s, hk, d), (s, hk, d), (t, h, d))]


@pytest.mark.parametrize("causal", [False, True], ids=["all", "causal"])
def test_attention_against_torch(causal):
    lengths, keys, h, hk, d = [5, 0, 9, 1], [5, 3, 14, 6], 6, 2, 8
    off, koff = np.cumsum([0, *lengths]), np.cumsum([0, *keys])
    q, k, v, g = _inputs(0, off[-1], koff[-1], h, hk, d)
    seqs = PA.sequences(off, koff)
    tq, tk, tv = (torch.from_numpy(x).requires_grad_(True) for x in (q, k, v))
    parts = []
    for q0, n, k0, m in seqs:
        kk, vv = (x[k0:k0 + m].repeat_interleave(h // hk, 1).transpose(0, 1) for x in (tk, tv))
        mask = torch.ones(n, m, dtype=torch.bool).tril(m - n) if causal else None
        parts.append(torch.nn.functional.scaled_dot_product_attention(tq[q0:q0 + n].transpose(0, 1), kk, vv, attn_mask=mask).transpose(0, 1))
    out = torch.cat(parts)
    out.backward(torch.from_numpy(g))
    np.testing.assert_allclose(PA.attention(q, k, v, seqs, causal), out.detach().numpy(), rtol=1e-12, atol=1e-12)
    for want, t in zip(PA.attention_vjp(q, k, v, g, seqs, causal), (tq, tk, tv)):
        np.testing.assert_allclose(want, t.grad.numpy(), rtol=1e-11, atol=1e-12)


def test_gradient_against_differences():
    """A central difference along a random direction; its error is of the third order, 1e-10 at a step of 1e-5."""
    off, koff = np.array([0, 7, 7, 12]), np.array([0, 4, 9, 20])
    q, k, v, g = _inputs(1, 12, 20, 4, 2, 8)
    seqs = PA.sequences(off, koff, [4, 5, 9])  # rows 0..2 of the first see no key; two rows of the last range are not keys
    grads = PA.attention_vjp(q, k, v, g, seqs)
    rng = np.random.default_rng(2)
    for i in range(3):
        step = rng.standard_normal((q, k, v)[i].shape)
        moved = [[x + (s * 1e-5 * step if j == i else 0) for j, x in enumerate((q, k, v))] for s in (1, -1)]
        slope = ((PA.attention(*moved[0], seqs) - PA.attention(*moved[1], seqs)) * g).sum() / 2e-5
        assert abs(slope - (grads[i] * step).sum()) <= 1e-8 * max(1.0, abs(slope))
    assert not grads[0][:3].any() and not PA.attention(q, k, v, seqs)[:3].any() and not grads[1][18:].any()


def test_known_answers_and_planted_mistakes():
    q, k, v, _ = _inputs(3, 6, 6, 2, 1, 8)
    off = np.array([0, 2, 6])
    seqs = PA.sequences(off)
    out = PA.attention(q, k, v, seqs)
    np.testing.assert_allclose(out[[0, 2]], v[[0, 2]].repeat(2, 1), rtol=1e-14)  # a first token sees itself
    np.testing.assert_allclose(PA.attention(0 * q, k, v, seqs, causal=False)[2:], np.broadcast_to(v[2:].mean(0), (4, 2, 8)), rtol=1e-14)
    for wrong in (PA.attention(q, k, v, seqs, causal=False), PA.attention(q, k, v, PA.sequences([0, 6])), PA.attention(q, k, v, seqs, scale=1.0)):
        assert np.abs(wrong - out).max() > 1e-2


@pytest.mark.parametrize("shared", [False, True])
@pytest.mark.parametrize("interleaved", [False, True])
def test_rotation_against_matrices(interleaved, shared):
    rng = np.random.default_rng(4)
    sections, d = (2, 1, 3), 14
    x, pos = rng.standard_normal((5, 3, d)), rng.integers(0, 50, (5, 3))
    got = RO.rotate(x, pos, sections, 100.0, shared, interleaved)
    for t in range(5):
        r = np.eye(d)
        i = 0
        for a, count in enumerate(sections):
            for j in range(count):
                angle = pos[t, a] / 100.0 ** (i / 6 if shared else j / count)
                u, w = (2 * i, 2 * i + 1) if interleaved else (i, i + 6)
                r[[u, u, w, w], [u, w, u, w]] = np.cos(angle), -np.sin(angle), np.sin(angle), np.cos(angle)
                i += 1
        np.testing.assert_allclose(got[t], x[t] @ r.T, rtol=1e-12, atol=1e-12)
        np.testing.assert_allclose(RO.rotate(x, pos, sections, 100.0, shared, interleaved, -1.0)[t], x[t] @ r, rtol=1e-12, atol=1e-12)
    # a score depends on the difference of the positions only
    y = rng.standard_normal((5, 3, d))
    a = (got * RO.rotate(y, pos + 3, sections, 100.0, shared, interleaved)).sum(-1)
    b = (RO.rotate(x, pos + 70, sections, 100.0, shared, interleaved) * RO.rotate(y, pos + 73, sections, 100.0, shared, interleaved)).sum(-1)
    np.testing.assert_allclose(a, b, rtol=1e-10, atol=1e-10)
