"""Packed attention with shaped scores on an MI355X: learned slopes, places past 2^24, parts of a call that another part
outweighs. Tolerances are the oracle's ``bounds``."""

from __future__ import annotations

import sys

import numpy as np
import pytest
import torch

from oracle import packed_attention_ref as PA
from oracle import shaped_attention_ref as SA
from rfdetr_jax_amd import _native, packed_attention

pytestmark = pytest.mark.gpu
HALF_STEP = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}
TYPES = pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])


def _dev():
    assert torch.cuda.is_available(), "GPU tests need a visible MI355X"
    return torch.device("cuda:0")


def _int(x):
    return torch.tensor([int(i) for i in x], dtype=torch.int32, device=_dev())


def _np(t):
    return t.detach().double().cpu().numpy()


def _normal(seed, dtype, *shapes):
    g = torch.Generator().manual_seed(seed)
    return [torch.randn(s, generator=g).to(dtype).to(_dev()) for s in shapes]


def _within(got, want, bound, what):
    got = _np(got)
    assert got.shape == want.shape and np.isfinite(got).all(), f"{what}: not finite"
    over = np.abs(got - want) - bound
    at = np.unravel_index(np.argmax(over), over.shape)
    assert over[at] <= 0, f"{what}: off by {abs(got[at] - want[at]):.3e} at {at}, {bound[at]:.3e} allowed"


@pytest.mark.parametrize("path", ["binding", "python"])
def test_learned_slopes_are_refused(path, monkeypatch):
    q, k, v = _normal(1, torch.bfloat16, (9, 4, 64), (9, 2, 64), (9, 2, 64))
    slopes = torch.nn.Parameter(torch.full((4,), 0.5, device=_dev()))
    if path == "python":
        monkeypatch.setattr(_native, "binding", lambda: _native._NoBinding)
    want = packed_attention(q, k, v, _int([0, 9]), slopes=slopes.detach())
    for x in (q, q.detach().requires_grad_(True)):
        with pytest.raises(ValueError, match="slopes get no gradient"):
            packed_attention(x, k, v, _int([0, 9]), slopes=slopes)
        with torch.no_grad():
            assert torch.equal(packed_attention(x, k, v, _int([0, 9]), slopes=slopes), want)


@TYPES
@pytest.mark.parametrize("dim", [8, 40])
def test_distances_past_2_to_the_24(dim, dtype):
    """The newest queries of a sequence of more than 2^24 keys, inside a window: their distances are small whole numbers,
    and their place is one that a float does not hold. What lies before the window holds NaN and is not seen."""
    m, n, h, window, tail = (1 << 24) + 301, 5, 2, 70, 200
    sys.stderr.write(f"[gpu] distances past 2^24, {dim} channels {dtype}\n")
    q, kt, vt, g = _normal(2, dtype, (n, h, dim), (tail, 1, dim), (tail, 1, dim), (n, h, dim))
    k, v = (torch.cat([torch.full((m - tail, 1, dim), float("nan"), dtype=dtype, device=_dev()), x]).requires_grad_(True) for x in (kt, vt))
    slopes = torch.tensor([1.0, 0.37], device=_dev())
    q.requires_grad_(True)
    for kw in (dict(), dict(cap=3.0), dict(cap=3.0, causal=False), dict(causal=False)):
        out = packed_attention(q, k, v, _int([0, n]), _int([0, m]), slopes=slopes, window=window, **kw)
        grads = torch.autograd.grad(out, (q, k, v), g)
        shape = SA.Shape(kw.get("causal", True), None, kw.get("cap"), _np(slopes), window)
        arrays, seqs = [_np(x) for x in (q, kt, vt, g)], PA.sequences([0, n], [0, tail])
        want = [SA.attention(*arrays[:3], seqs, shape), *SA.attention_vjp(*arrays, seqs, shape)]
        got = [out, grads[0], grads[1][-tail:], grads[2][-tail:]]
        for name, x, w, b in zip(("out", "grad_q", "grad_k", "grad_v"), got, want, SA.bounds(*arrays, seqs, HALF_STEP[dtype], shape)):
            _within(x, w, b, f"{name} {kw}")
        assert not grads[1][:-tail].any() and not grads[2][:-tail].any()


@TYPES
@pytest.mark.parametrize("n", [1, 20], ids=["token", "chunk"])
@pytest.mark.parametrize("value", [float("nan"), float("inf")])
def test_a_value_that_is_not_finite_in_a_part_that_weighs_nothing(value, n, dtype):
    """Slopes so steep that the first keys weigh 0 beside the last: a value of theirs that is not finite shows in the rows
    that see it, whichever workgroup took it, and in its channel alone."""
    m, h, hk, d = 5000, 4, 2, 64
    q, k, v = _normal(3, dtype, (n, h, d), (m, hk, d), (m, hk, d))
    slopes = torch.full((h,), 0.5, device=_dev())
    want = packed_attention(q, k, v, _int([0, n]), _int([0, m]), slopes=slopes)
    for key in (10, 2600):
        odd = v.clone()
        odd[key, 1, 33] = value
        got = packed_attention(q, k, odd, _int([0, n]), _int([0, m]), slopes=slopes)
        assert not torch.isfinite(got[:, 2:, 33]).any()
        rest = [c for c in range(d) if c != 33]
        assert torch.equal(got[:, 2:, rest], want[:, 2:, rest]) and torch.equal(got[:, :2], want[:, :2])


@TYPES
@pytest.mark.parametrize("kw", [{}, dict(cap=4.0), dict(window=250), dict(window=100)], ids=["plain", "cap", "window", "narrow"])
def test_values_that_are_not_finite_at_both_ends_of_what_a_row_sees(kw, dtype):
    """Two values of one channel that are not finite, one in a chunk that every row of the workgroup sees and one on the
    diagonal or at the window's end: the rows that see both get their sum, those that see one get it."""
    n, h, hk, d = 400, 4, 2, 64
    q, k, v = _normal(4, dtype, (n, h, d), (n, hk, d), (n, hk, d))
    q = 0.1 * q  # every weight is well above 0
    clean = packed_attention(q, k, v, _int([0, n]), **kw)
    inf, nan = float("inf"), float("nan")
    places = torch.arange(n, device=_dev())

    def sees(key):
        return (places >= key) & (places - key < kw.get("window", n))

    for first, last, a, b in ((20, 300, inf, -inf), (20, 300, nan, inf), (140, 390, -inf, inf), (200, 270, inf, -inf), (20, 300, inf, inf)):
        odd = v.clone()
        odd[first, :, 5], odd[last, :, 5] = a, b
        got = packed_attention(q, k, odd, _int([0, n]), **kw)
        both, one, other = sees(first) & sees(last), sees(first) & ~sees(last), sees(last) & ~sees(first)
        for rows, value in ((both, a + b), (one, a), (other, b)):
            x = got[rows][..., 5].float()
            assert torch.isnan(x).all() if value != value else (x == value).all(), (first, last, a, b, value)
        none = ~(sees(first) | sees(last))
        assert torch.equal(got[none], clean[none])
        rest = [c for c in range(d) if c != 5]
        assert torch.equal(got[..., rest], clean[..., rest])


@TYPES
@pytest.mark.parametrize("kw", [{}, dict(cap=4.0), dict(window=100), dict(window=30, cap=4.0), dict(window=90, causal=False)],
                         ids=["plain", "cap", "window", "narrow", "open"])
@pytest.mark.parametrize("dim", [64, 128])
def test_chunk_after_chunk_of_values_that_are_not_finite(dim, kw, dtype):
    """Values that are not finite in every chunk on a tile's diagonal and at its window's ends, one chunk behind the other:
    each is searched and settled before any wave multiplies with it. Rows that see none of them keep their bits, in call
    after call, and those that see one have NaN in its channel alone."""
    n, h, hk = 700, 2, 2
    q, k, v = _normal(5, dtype, (n, h, dim), (n, hk, dim), (n, hk, dim))
    off, window, causal = _int([0, n]), kw.get("window", n), kw.get("causal", True)
    clean = packed_attention(q, k, v, off, **kw)
    keys = list(range(40, n, 61))
    odd = v.clone()
    odd[keys, :, 7] = float("nan")
    odd[keys, :, dim - 3] = float("nan")
    place, key = torch.arange(n, device=_dev())[:, None], torch.tensor(keys, device=_dev())[None]
    sees = ((place - key).abs() < window) & ((key <= place) if causal else torch.ones_like(key <= place))
    sees = sees.any(1)
    rest = [c for c in range(dim) if c not in (7, dim - 3)]
    for _ in range(10):
        got = packed_attention(q, k, odd, off, **kw)
        assert torch.equal(got[~sees], clean[~sees])
        assert torch.isnan(got[sees][..., [7, dim - 3]]).all()
        assert torch.equal(got[sees][..., rest], clean[sees][..., rest])
