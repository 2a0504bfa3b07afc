"""The oracle of packed attention with shaped scores, against torch's float64 autograd, central differences and the
oracle of the plain one, and planted mistakes."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import packed_attention_ref as PA
from oracle import shaped_attention_ref as SA

OFF, KOFF = [0, 9, 9, 30], [2, 15, 20, 44]
SEQS = PA.sequences(OFF, KOFF)
OPTIONS = {
    "cap": dict(cap=1.5), "slopes": dict(slopes=[0.5, 0.03]), "window": dict(window=4), "prefix": dict(prefixes=[6, 2, 30]),
    "all": dict(cap=3.0, slopes=[0.25, -0.1], window=7, prefixes=[5, 0, 17]), "both_sides": dict(causal=False, window=3, slopes=[1.0, 0.1]),
}


def _arrays(seed=0):
    r = np.random.default_rng(seed)
    return r.standard_normal((31, 2, 8)), *(r.standard_normal((44, 1, 8)) for _ in range(2)), r.standard_normal((31, 2, 8))


def _torch(q, k, v, grad, shape):
    at = [torch.tensor(x, requires_grad=True) for x in (q, k, v)]
    out = torch.zeros(q.shape, dtype=torch.float64)
    for i, (q0, n, k0, m) in enumerate(SEQS):
        for h in range(2 if n and m else 0):
            x = at[0][q0:q0 + n, h] @ at[1][k0:k0 + m, 0].T / 8 ** 0.5
            if shape.cap is not None:
                x = shape.cap * torch.tanh(x / shape.cap)
            for t in range(n):
                see = []
                for j in range(m):
                    place = t + m - n
                    ok = not shape.causal or j <= place or (shape.prefixes is not None and j < shape.prefixes[i])
                    if ok and (shape.window is None or abs(place - j) < shape.window):
                        see.append(j)
                if see:
                    away = torch.tensor([abs(t + m - n - j) for j in see], dtype=torch.float64)
                    row = x[t, see] - (0.0 if shape.slopes is None else shape.slopes[h] * away)
                    out[q0 + t, h] = torch.softmax(row, 0) @ at[2][k0:k0 + m, 0][see]
    grads = torch.autograd.grad(out, at, torch.tensor(grad))
    return [x.detach().numpy() for x in (out, *grads)]


@pytest.mark.parametrize("name", sorted(OPTIONS))
def test_against_autograd(name):
    arrays, shape = _arrays(), SA.Shape(**OPTIONS[name])
    got = [SA.attention(*arrays[:3], SEQS, shape), *SA.attention_vjp(*arrays, SEQS, shape)]
    for x, w in zip(got, _torch(*arrays, shape)):
        np.testing.assert_allclose(x, w, rtol=0, atol=1e-12)


def test_without_a_shape_it_is_the_plain_attention():
    arrays = _arrays(1)
    for causal in (True, False):
        got = [SA.attention(*arrays[:3], SEQS, SA.Shape(causal)), *SA.attention_vjp(*arrays, SEQS, SA.Shape(causal))]
        want = [PA.attention(*arrays[:3], SEQS, causal), *PA.attention_vjp(*arrays, SEQS, causal)]
        for x, w in zip(got, want):
            np.testing.assert_allclose(x, w, rtol=0, atol=1e-13)


@pytest.mark.parametrize("name", sorted(OPTIONS))
def test_gradients_against_differences(name):
    arrays, shape, r = _arrays(2), SA.Shape(**OPTIONS[name]), np.random.default_rng(3)
    grads = SA.attention_vjp(*arrays, SEQS, shape)
    for i in range(3):
        way, h = r.standard_normal(arrays[i].shape), 1e-6
        ends = []
        for sign in (1, -1):
            moved = list(arrays)
            moved[i] = moved[i] + sign * h * way
            ends.append((SA.attention(*moved[:3], SEQS, shape) * arrays[3]).sum())
        assert abs((ends[0] - ends[1]) / (2 * h) - (grads[i] * way).sum()) < 1e-7 * (1 + np.abs(grads[i] * way).sum())


@pytest.mark.parametrize("mistake", ["slope_before_cap", "window_one_off", "no_bend", "prefix_of_another"])
def test_planted_mistakes_leave_the_bounds(mistake):
    """What a kernel might get wrong is outside the bounds, even those of bf16."""
    arrays = _arrays(4)
    shape = SA.Shape(**OPTIONS["all"])
    want = [SA.attention(*arrays[:3], SEQS, shape), *SA.attention_vjp(*arrays, SEQS, shape)]
    other = dict(OPTIONS["all"])
    if mistake == "window_one_off":
        other["window"] = 8
    elif mistake == "prefix_of_another":
        other["prefixes"] = [0, 17, 5]
    wrong = SA.Shape(**other)
    if mistake == "slope_before_cap":
        right = wrong.scores

        def scores(q, k, head, seq):
            s, t, x, away, seen = right(q, k, head, seq)
            return s, t, wrong.cap * np.tanh((s - away) / wrong.cap), away, seen

        wrong.scores = scores
    elif mistake == "no_bend":
        right = wrong.scores
        wrong.scores = lambda q, k, head, seq: (lambda s, t, x, away, seen: (s, np.zeros_like(t), x, away, seen))(*right(q, k, head, seq))
    got = [SA.attention(*arrays[:3], SEQS, wrong), *SA.attention_vjp(*arrays, SEQS, wrong)]
    bound = SA.bounds(*arrays, SEQS, 2.0 ** -8, shape)
    assert any((np.abs(g - w) > b).any() for g, w, b in zip(got, want, bound))
