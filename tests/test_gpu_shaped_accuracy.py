"""Packed attention in bf16 on an MI355X: how far the gradients' norms are off, with shaped scores and without, where errors
average out least. The tolerances follow from which numbers are rounded to bf16, and how often."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import packed_attention_ref as PA
from oracle import shaped_attention_ref as SA
from rfdetr_jax_amd import packed_attention

pytestmark = pytest.mark.gpu
HALF_STEP = 2.0 ** -8


def _dev():
    assert torch.cuda.is_available(), "GPU tests need a visible MI355X"
    return torch.device("cuda:0")


def _np(t):
    return t.detach().double().cpu().numpy()


def _rounded(x):
    """The norm of what rounding ``x`` to bf16 takes from it."""
    return np.linalg.norm(_np(torch.from_numpy(x).bfloat16()) - x)


def _made(seed, n, h, hk, dim, sharp=1.0):
    g = torch.Generator().manual_seed(seed)
    return [(f * torch.randn(n, heads, dim, generator=g)).bfloat16().to(_dev()) for heads, f in ((h, sharp), (hk, 1.0), (hk, 1.0), (h, 1.0))]


def _run(q, k, v, g, off, **kw):
    leaves = [x.detach().requires_grad_(True) for x in (q, k, v)]
    out = packed_attention(*leaves, torch.tensor(off, dtype=torch.int32, device=_dev()), **kw)
    return (out, *torch.autograd.grad(out, leaves, g))


@pytest.mark.parametrize("dim, cap", [(96, 50.0), (128, 50.0), (64, None), (80, None), (96, None), (128, None)])
def test_sharp_scores_of_many_channels(dim, cap):
    """Scores of four standard deviations where ds is rounded once. The keys that a row weighs most share up to a = 4 standard
    deviations along its query. That part cancels in the sum of ds k, and not in the sum of the roundings of ds times k: this
    is the result's own rounding times the root of (a^2 + D) / D, and both together the root of 1 + (a^2 + D) / D of it."""
    n, h, hk = 900, 4, 2
    q, k, v, g = _made(31 + dim, n, h, hk, dim, 4.0)
    shape = SA.Shape(cap=cap, window=None if cap else n)
    got = _run(q, k, v, g, [0, n], cap=cap, window=shape.window)
    want = SA.attention_vjp(*(_np(x) for x in (q, k, v, g)), PA.sequences([0, n]), shape)
    most = (1 + (16 + dim) / dim) ** 0.5
    assert np.linalg.norm(_np(got[1]) - want[0]) <= most * _rounded(want[0])


KINDS = {"plain": {}, "cap": dict(cap=5.0), "slopes": dict(slopes=0.5), "window": dict(window=5), "all": dict(cap=2.0, slopes=0.25, window=7)}


@pytest.mark.parametrize("n, kind", [(n, kind) for n in (2, 4, 8, 16, 31) for kind in sorted(KINDS)] + [(90, "window"), (90, "all")])
@pytest.mark.parametrize("dim", [32, 128])
def test_few_tokens_and_narrow_windows(n, kind, dim):
    """out and grad_q keep what the rounding of the weights and of ds leaves where rows see fewer than 64 keys. grad_k and grad_v take them rounded once, by up to half a step each,
    and so few errors need not average out. So with w for the weights, ds for their gradients, and r what is rounded away of
    the exact result, the norms are off by at most
        out, grad_q: |r|,     grad_v: |r| + u |w^T |g||,     grad_k: |r| + u scale | |ds|^T |q| |
    (the inner norms over channels), besides 2^-14 of what the f32 sums add up."""
    h, hk, off = 4, 2, [0, n]
    q, k, v, g = _made(7 * n + dim, n, h, hk, dim)
    kw = dict(KINDS[kind])
    if "slopes" in kw:
        kw["slopes"] = torch.tensor([kw["slopes"] * 0.7 ** i for i in range(h)], device=_dev())
    shape = SA.Shape(cap=kw.get("cap"), window=kw.get("window"), slopes=_np(kw["slopes"]) if "slopes" in kw else None)
    got = _run(q, k, v, g, off, **kw)
    arrays = [_np(x) for x in (q, k, v, g)]
    want = [SA.attention(*arrays[:3], PA.sequences(off), shape), *SA.attention_vjp(*arrays, PA.sequences(off), shape)]
    scale = dim ** -0.5
    once, sums = {2: np.zeros((n, hk)), 3: np.zeros((n, hk))}, [np.zeros((n, h)), np.zeros((n, h)), np.zeros((n, hk)), np.zeros((n, hk))]
    norm = [np.linalg.norm(x, axis=-1) for x in arrays]
    for head in range(h):
        b = head // (h // hk)
        _, t, x, _, seen = shape.scores(arrays[0][:, head], arrays[1][:, b], head, 0)
        p = SA._softmax(x, seen)[0]
        dp = arrays[3][:, head] @ arrays[2][:, b].T
        ds = p * (dp - (p * dp).sum(-1, keepdims=True)) * (1 - t * t) * scale
        once[2][:, b] += np.abs(ds).T @ norm[0][:, head]
        once[3][:, b] += p.T @ norm[3][:, head]
        most = scale * p * norm[3][:, head][:, None] * norm[2][:, b].max()
        sums[0][:, head] = p @ norm[2][:, b]
        sums[1][:, head] = most @ norm[1][:, b]
        sums[2][:, b] += most.T @ norm[0][:, head]
        sums[3][:, b] += p.T @ norm[3][:, head]
    for i, name in enumerate(("out", "grad_q", "grad_k", "grad_v")):
        allowed = _rounded(want[i]) + 2.0 ** -14 * np.linalg.norm(sums[i])
        if i >= 2:
            allowed += HALF_STEP * np.linalg.norm(once[i])
        off_by = np.linalg.norm(_np(got[i]) - want[i])
        assert off_by <= allowed, f"{name}: off by {off_by:.3e}, {allowed:.3e} allowed"
