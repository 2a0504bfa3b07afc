"""Rotary positions on several axes (msda_rotary through rfdetr_jax_amd.rotary_embed) on an MI355X, against the
float64 oracle.

Tolerance, element by element: the angle is reduced in f64 and rounded once in [-1/2, 1/2] turns (pi 2^-25 of
an angle), cos and sin have a few units in the last place (4 2^-24 taken), each product and the sum round
once (2 2^-24): 8 2^-24 of |u| + |w|, and half a step of the type for the result.
"""

from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import rotary_ref as RO
from rfdetr_jax_amd import rotary_embed

pytestmark = pytest.mark.gpu
HALF_STEP = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}
TYPES = pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])


def _dev():
    assert torch.cuda.is_available(), "GPU tests need a visible MI355X"
    return torch.device("cuda:0")


def _np(t):
    return t.detach().double().cpu().numpy()


def _normal(seed, dtype, *shapes):
    g = torch.Generator().manual_seed(seed)
    return [torch.randn(s, generator=g).to(dtype).to(_dev()) for s in shapes]


def _check(got, x, pos, sections, base=10000.0, shared=False, interleaved=False, sign=1.0):
    x64, p = _np(x), pos.cpu().numpy()
    want = RO.rotate(x64, p, sections, base, shared, interleaved, sign)
    n = sum(sections)
    a, b = (slice(0, 2 * n, 2), slice(1, 2 * n, 2)) if interleaved else (slice(0, n), slice(n, 2 * n))
    bound = HALF_STEP[x.dtype] * np.abs(want)
    for s in (a, b):
        bound[..., s] += 8 * 2.0 ** -24 * (np.abs(x64[..., a]) + np.abs(x64[..., b]))
    bound[..., 2 * n:] = 0  # passes unchanged
    over = np.abs(_np(got) - want) - bound
    assert got.dtype == x.dtype and over.max() <= 0, f"{over.max():.3e} past the bound"


#      tokens, heads, key heads, head dim, sections
SHAPES = {
    "token": (1, 8, 2, 64, (32,)),
    "three_axes": (700, 4, 1, 128, (16, 24, 24)),
    "many_tokens": (9001, 2, 1, 64, (12, 20)),
    "part": (33, 3, 3, 80, (8, 8)),             # channels 32 .. 79 pass
    "odd_sections": (65, 2, 1, 72, (5, 7, 1)),  # no whole pieces
    "eight_axes": (10, 1, 1, 32, (1, 2, 3, 1, 1, 1, 4, 3)),
    "dim2": (5, 1, 1, 2, (1,)),
    "dim256": (20, 2, 1, 256, (64, 64)),
}


@TYPES
@pytest.mark.parametrize("interleaved", [False, True], ids=["halves", "neighbours"])
@pytest.mark.parametrize("name", sorted(SHAPES))
def test_against_oracle(name, interleaved, dtype):
    t, h, hk, d, sections = SHAPES[name]
    q, k, gq, gk = _normal(1, dtype, (t, h, d), (t, hk, d), (t, h, d), (t, hk, d))
    rng = np.random.default_rng(2)
    for shared, pos in ((True, torch.from_numpy(rng.integers(0, 2_000_000, (t, len(sections))).astype(np.int32))),
                        (False, torch.from_numpy(rng.integers(-(1 << 40), 1 << 40, (t, len(sections))))),
                        (False, torch.from_numpy((rng.random((t, len(sections))) * 40).astype(np.float32)))):
        pos = pos.to(_dev())
        leaves = [x.detach().requires_grad_(True) for x in (q, k)]
        outs = rotary_embed(*leaves, pos, sections, shared_frequencies=shared, interleaved=interleaved)
        grads = torch.autograd.grad(outs, leaves, (gq, gk))
        if pos.dtype == torch.int64:
            # a frequency's own f64 rounding (2^-53 relative, a few steps) times a position of 2^40: 2^-11 of a turn
            for got, x in zip((*outs, *grads), (q, k, gq, gk)):
                assert torch.isfinite(got).all()
                np.testing.assert_allclose((_np(got) ** 2).sum(-1), (_np(x) ** 2).sum(-1), rtol=4 * HALF_STEP[dtype] + 2.0 ** -18)
            continue
        for got, x, sign in ((outs[0], q, 1.0), (outs[1], k, 1.0), (grads[0], gq, -1.0), (grads[1], gk, -1.0)):
            _check(got, x, pos, sections, shared=shared, interleaved=interleaved, sign=sign)


@TYPES
def test_leading_axes_strides_and_single_tensors(dtype):
    """[B, T, H, D] slices of one projection, positions with the axes first, no k, one gradient only, a cotangent by stride
    0, rows off their 16-byte boundaries."""
    (qkv,) = _normal(3, dtype, (2, 50, 6, 64))
    pos = torch.randint(0, 99, (3, 2, 50), device=_dev()).movedim(0, -1)
    sections = (8, 8, 16)
    q, k = rotary_embed(qkv[:, :, :4], qkv[:, :, 4:5], pos, sections)
    _check(q, qkv[:, :, :4], pos, sections)
    _check(k, qkv[:, :, 4:5], pos, sections)
    assert torch.equal(rotary_embed(qkv[:, :, :4], None, pos, sections), q)
    shifted = torch.empty(qkv.numel() + 1, dtype=dtype, device=_dev())[1:].view(qkv.shape).copy_(qkv)
    got = rotary_embed(shifted[:, :, :4], shifted[:, :, 4:5], pos, sections)
    assert torch.equal(got[0], q) and torch.equal(got[1], k)
    assert torch.equal(rotary_embed(qkv[0, 0, :4], None, pos[0, 0], sections), q[0, 0])
    channels = qkv.transpose(2, 3).contiguous().transpose(2, 3)
    assert torch.equal(rotary_embed(channels, None, pos, sections)[:, :, :4], q)
    leaf = qkv.detach().requires_grad_(True)
    outs = rotary_embed(leaf[:, :, :4], leaf[:, :, 4:], pos, sections)
    (grad,) = torch.autograd.grad(outs[1].sum(), leaf)
    assert not grad[:, :, :4].any()
    _check(grad[:, :, 4:], torch.ones_like(qkv[:, :, 4:]), pos, sections, sign=-1.0)
    for shape in ((0, 4, 64), (2, 0, 4, 64), (3, 0, 64)):
        x = torch.empty(shape, dtype=dtype, device=_dev())
        p = torch.zeros((*shape[:-2], 3), dtype=torch.int32, device=_dev())
        assert rotary_embed(x, x, p, sections)[0].shape == x.shape


def test_far_positions_keep_their_difference():
    """The product of a turned query and key depends on the difference of their positions: moved by 2^30, within the
    tolerance of the two rotations (twice 8 2^-24 of the row's squared length) and 2^-20 for the f64 frequency times 2^30."""
    q, k = _normal(4, torch.float32, (64, 1, 64), (64, 1, 64))
    p = torch.arange(64, dtype=torch.int64, device=_dev())[:, None]
    near, far = (tuple(rotary_embed(x, None, p + s, (32,)).double() for x, s in ((q, a), (k, a + 5))) for a in (0, 1 << 30))
    a, b = (near[0] * near[1]).sum(-1), (far[0] * far[1]).sum(-1)
    reach = q.double().norm(dim=-1) * k.double().norm(dim=-1)
    assert ((a - b).abs() <= (32 * 2.0 ** -24 + 2.0 ** -20) * reach).all()


@TYPES
def test_in_a_graph(dtype):
    q, k, g = _normal(5, dtype, (90, 4, 64), (90, 2, 64), (90, 4, 64))
    pos = torch.randint(0, 1000, (90, 2), device=_dev(), dtype=torch.int32)

    def work():
        return rotary_embed(q, k, pos, (16, 16), interleaved=True)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        work()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        outs = work()
    for _ in range(3):
        pos.add_(37)
        q.mul_(-0.5)
        eager = work()
        torch.cuda.synchronize()
        for x in outs:
            x.fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, eager))


def test_refusals_and_second_derivatives():
    q, pos = torch.randn(6, 2, 32, device=_dev()), torch.zeros(6, 2, dtype=torch.int32, device=_dev())
    for args, error, text in (
            ((q.double(), None, pos, (8, 8)), TypeError, "not supported"), ((q[0, 0], None, pos, (8, 8)), ValueError, "heads, D"),
            ((q, q.bfloat16(), pos, (8, 8)), TypeError, "one type"), ((q, q[:5], pos, (8, 8)), ValueError, "expected"), ((q, q[..., :16], pos, (4, 4)), ValueError, "expected"),
            ((q, q, pos.to(torch.int16), (8, 8)), TypeError, "int32"), ((q, q, pos.cpu(), (8, 8)), ValueError, "cpu"), ((q, q, pos, (8, 8, 1)), ValueError, "positions"),
            ((q, q, pos, ()), ValueError, "sections"), ((q, q, pos, (8, 0)), ValueError, "sections"), ((q, q, pos, (8, 9)), ValueError, "pairs"),
            ((q[..., :31], None, pos, (8, 7)), ValueError, "even"), ((q, q, pos, (8, 8), 0.0), ValueError, "base"), ((q, q, pos, (8, 8), float("inf")), ValueError, "base"),
            ((q.cpu(), None, pos, (8, 8)), RuntimeError, "no CPU path")):
        with pytest.raises(error, match=text):
            rotary_embed(*args)
    leaf, g = q.clone().requires_grad_(True), torch.randn_like(q).requires_grad_(True)
    (grad,) = torch.autograd.grad(rotary_embed(leaf, None, pos, (8, 8)), [leaf], g, create_graph=True)
    with pytest.raises(RuntimeError, match="differentiate"):
        torch.autograd.grad(grad.sum(), [leaf])


@TYPES
@pytest.mark.parametrize("interleaved", [False, True], ids=["halves", "neighbours"])
def test_int64_positions_past_32_bits_against_oracle(interleaved, dtype):
    """Positions of 2^33 to 2^36 of either sign, whose low 32 bits are other positions. Beside the usual bound an angle is
    off by its f64 steps: a frequency base ** -e is formed from a rounded exponent, e ln(base) < 9.3, so that two ways to
    it differ by 4 roundings of at most 9.3 and 8 of 1, less than 2^6 times 2^-53; that relative error of an angle
    moves a channel by |angle| 2^-47 of |u| + |w|. At 2^36 it is 2^-11, at the low 32 bits' angle or the other sign
    of the order of 1."""
    sections = (8, 12, 12)
    q, k, gq, gk = _normal(6, dtype, (150, 2, 64), (150, 1, 64), (150, 2, 64), (150, 1, 64))
    rng = np.random.default_rng(7)
    pos = (rng.choice([-1, 1], (150, 3)) * np.exp2(rng.uniform(33, 36, (150, 3)))).astype(np.int64)
    p = torch.from_numpy(pos).to(_dev())
    for shared in (False, True):
        leaves = [x.detach().requires_grad_(True) for x in (q, k)]
        outs = rotary_embed(*leaves, p, sections, shared_frequencies=shared, interleaved=interleaved)
        grads = torch.autograd.grad(outs, leaves, (gq, gk))
        angle = np.abs(RO.angles(pos, sections, shared=shared))[:, None]
        for got, x, sign in ((outs[0], q, 1.0), (outs[1], k, 1.0), (grads[0], gq, -1.0), (grads[1], gk, -1.0)):
            x64 = _np(x)
            want = RO.rotate(x64, pos, sections, 10000.0, shared, interleaved, sign)
            a, b = (slice(0, 64, 2), slice(1, 64, 2)) if interleaved else (slice(0, 32), slice(32, 64))
            reach = np.abs(x64[..., a]) + np.abs(x64[..., b])
            for s in (a, b):
                bound = HALF_STEP[dtype] * np.abs(want[..., s]) + (8 * 2.0 ** -24 + angle * 2.0 ** -47) * reach
                assert (np.abs(_np(got)[..., s] - want[..., s]) <= bound * (1 + HALF_STEP[dtype])).all()
            # positions cut to 32 bits, or of the other sign, are far outside
            for wrong in (pos.astype(np.int32), -pos):
                other = RO.rotate(x64, wrong, sections, 10000.0, shared, interleaved, sign)
                assert np.abs(_np(got) - other).max() > 0.5
