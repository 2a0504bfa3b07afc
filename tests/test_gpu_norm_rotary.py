"""Norms of queries and keys with rotary positions (rfdetr_jax_amd.norm_rotary_embed) on an MI355X, against the float64
oracle, element by element within its bounds."""

from __future__ import annotations

import sys

import numpy as np
import pytest
import torch

from oracle import norm_rotary_ref as NR
from oracle import shaped_attention_ref as SA
from rfdetr_jax_amd import _native, norm_rotary_embed, packed_attention

pytestmark = pytest.mark.gpu
HALF_STEP = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}
TYPES = pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])


def _dev():
    assert torch.cuda.is_available(), "GPU tests need a visible MI355X"
    return torch.device("cuda:0")


def _np(t):
    return None if t is None else t.detach().double().cpu().numpy()


def _normal(seed, dtype, *shapes):
    g = torch.Generator().manual_seed(seed)
    return [torch.randn(s, generator=g).to(dtype).to(_dev()) for s in shapes]


def _positions(t, axes, kind="int", seed=2):
    r = np.random.default_rng(seed)
    x = r.integers(0, 2_000_000, (t, axes)).astype(np.int32) if kind == "int" else (r.random((t, axes)) * 40).astype(np.float32)
    return torch.from_numpy(x).to(_dev())


def _within(got, want, bound, what):
    got = _np(got)
    assert got.shape == want.shape and np.isfinite(got).all(), what
    over = np.abs(got - want) - bound
    at = np.unravel_index(np.argmax(over), over.shape)
    assert over[at] <= 0, f"{what}: off by {abs(got[at] - want[at]):.3e} at {at}, {bound[at]:.3e} allowed"


def _run(q, k, qw, kw, pos, sections, gq, gk, **options):
    leaves = [None if x is None else x.detach().requires_grad_(True) for x in (q, k, qw, kw)]
    outs = norm_rotary_embed(*leaves, pos, sections, **options)
    outs = (outs,) if k is None else outs
    given = [x for x in leaves if x is not None]
    grads = iter(torch.autograd.grad(outs, given, (gq,) if k is None else (gq, gk)))
    return outs, [None if x is None else next(grads) for x in leaves]


def _check(outs, grads, q, k, qw, kw, pos, sections, gq, gk, eps=1e-6, **options):
    p, u = pos.reshape(-1, pos.shape[-1]).cpu().numpy(), HALF_STEP[q.dtype]
    options = {"shared": options.get("shared_frequencies", False), "interleaved": options.get("interleaved", False), "base": options.get("base", 10000.0)}
    flat = lambda t: _np(t).reshape(-1, *t.shape[-2:])  # noqa: E731
    for i, (x, w, g) in enumerate(((q, qw, gq), (k, kw, gk))):
        if x is None:
            continue
        assert outs[i].dtype == x.dtype and outs[i].shape == x.shape
        args = (flat(x), _np(w), p, sections, eps)
        _within(outs[i].reshape(-1, *x.shape[-2:]), NR.forward(*args, **options), NR.forward_bound(*args, u, **options), f"out {i}")
        args = (flat(x), _np(w), flat(g), p, sections, eps)
        dx, dw = NR.backward(*args, **options)
        bx, bw = NR.backward_bounds(*args, u, 0.0 if w is None else HALF_STEP[w.dtype], **options)
        if grads[i] is not None:
            assert grads[i].shape == x.shape and grads[i].dtype == x.dtype
            _within(grads[i].reshape(-1, *x.shape[-2:]), dx, bx, f"grad {i}")
        if w is not None and grads[2 + i] is not None:
            assert grads[2 + i].dtype == w.dtype
            _within(grads[2 + i], dw, bw, f"grad of weight {i}")


#      tokens, heads, key heads, head dim, sections
SHAPES = {
    "token": (1, 8, 2, 64, (32,)),
    "three_axes": (700, 4, 1, 128, (16, 24, 24)),
    "many_tokens": (9001, 2, 1, 64, (12, 20)),
    "persistent": (40001, 1, 1, 32, (16,)),     # more tokens than one round of the backward's workgroups
    "part": (33, 3, 3, 80, (8, 8)),             # channels 32 .. 79 are not turned
    "odd_rest": (33, 2, 1, 72, (8, 16)),        # an odd number of pieces behind the pairs
    "odd_sections": (65, 2, 1, 74, (5, 7, 1)),  # no whole pieces
    "eight_axes": (10, 1, 1, 32, (1, 2, 3, 1, 1, 1, 4, 3)),
    "dim2": (5, 1, 1, 2, (1,)),
    "dim256": (20, 2, 1, 256, (64, 64)),
    "dim256_little": (20, 2, 1, 256, (8,)),
}


@TYPES
@pytest.mark.parametrize("interleaved", [False, True], ids=["halves", "neighbours"])
@pytest.mark.parametrize("name", sorted(SHAPES))
def test_against_oracle(name, interleaved, dtype):
    t, h, hk, d, sections = SHAPES[name]
    sys.stderr.write(f"[gpu] norm rotary {name} {interleaved} {dtype}\n")
    q, k, gq, gk = _normal(1, dtype, (t, h, d), (t, hk, d), (t, h, d), (t, hk, d))
    q = q * 3
    for wt, kind, shared in ((torch.float32, "int", True), (torch.bfloat16, "float", False), (None, "int", False)):
        qw, kw = (None, None) if wt is None else (1 + 0.2 * x for x in _normal(3, wt, (d,), (d,)))
        pos = _positions(t, len(sections), kind)
        options = dict(shared_frequencies=shared, interleaved=interleaved)
        outs, grads = _run(q, k, qw, kw, pos, sections, gq, gk, **options)
        _check(outs, grads, q, k, qw, kw, pos, sections, gq, gk, **options)


@TYPES
def test_layouts(dtype):
    """[B, T, H, D] slices of one projection, no k, one weight alone, strides of 0, rows off their 16-byte boundaries,
    channels that are not contiguous: the same results."""
    b, t, h, hk, d, sections = 2, 17, 4, 2, 64, (20, 12)
    (qkv,) = _normal(4, dtype, (b, t, h + 2 * hk, d))
    q, k = qkv[:, :, :h], qkv[:, :, h:h + hk]
    gq, gk, qw, kw = _normal(5, dtype, (b, t, h, d), (b, t, hk, d), (d,), (d,))
    pos = _positions(b * t, 2).view(b, t, 2)
    outs, grads = _run(q, k, qw, kw, pos, sections, gq, gk)
    _check(outs, grads, q, k, qw, kw, pos, sections, gq, gk)
    shifted = [torch.empty(x.numel() + 1, dtype=dtype, device=_dev())[1:].view(x.shape).copy_(x) for x in (q, k)]
    channels = [x.transpose(-1, -2).contiguous().transpose(-1, -2) for x in (q, k)]
    for other, exact in ((shifted, False), (channels, True), ([x.contiguous() for x in (q, k)], True)):
        o2, g2 = _run(*other, qw, kw, pos, sections, gq, gk)
        _check(o2, g2, q, k, qw, kw, pos, sections, gq, gk)
        if exact:
            assert all(torch.equal(x, y) for x, y in zip((*outs, *grads), (*o2, *g2)))
    alone, g1 = _run(q, None, qw, None, pos, sections, gq, None)
    assert torch.equal(alone[0], outs[0]) and torch.equal(g1[0], grads[0]) and torch.equal(g1[2], grads[2])
    for qw1, kw1 in ((qw, None), (None, kw)):
        o, g = _run(q, k, qw1, kw1, pos, sections, gq, gk)
        _check(o, g, q, k, qw1, kw1, pos, sections, gq, gk)
    head = q[:, :, :1].expand(b, t, h, d)
    ones = torch.ones((), dtype=dtype, device=_dev()).expand(b, t, h, d)
    o, g = _run(head, k, qw, kw, pos, sections, ones, gk)
    _check(o, g, head, k, qw, kw, pos, sections, ones, gk)
    single, gs = _run(q[0, 0], k[0, 0], qw, kw, pos[0, 0], sections, gq[0, 0], gk[0, 0])  # one token, no leading axis
    assert torch.equal(single[0], outs[0][0, 0]) and torch.equal(gs[1], grads[1][0, 0])


@TYPES
def test_gradients_wanted_one_by_one(dtype):
    t, h, hk, d, sections = 50, 3, 2, 64, (32,)
    q, k, gq, gk, qw, kw = _normal(6, dtype, (t, h, d), (t, hk, d), (t, h, d), (t, hk, d), (d,), (d,))
    pos = _positions(t, 1)
    outs, want = _run(q, k, qw, kw, pos, sections, gq, gk)
    for i in range(4):
        leaves = [x.detach().requires_grad_(j == i) for j, x in enumerate((q, k, qw, kw))]
        out = norm_rotary_embed(*leaves, pos, sections)
        (grad,) = torch.autograd.grad(out, [leaves[i]], (gq, gk))
        assert torch.equal(grad, want[i]), i
    for which in range(2):  # a cotangent of one result only
        leaves = [x.detach().requires_grad_(True) for x in (q, k, qw, kw)]
        out = norm_rotary_embed(*leaves, pos, sections)
        grads = torch.autograd.grad(out[which], leaves, (gq, gk)[which], allow_unused=True)
        for i in range(4):
            assert torch.equal(grads[i], want[i]) if i % 2 == which else grads[i] is None
    with torch.no_grad():
        assert all(torch.equal(a, b) for a, b in zip(norm_rotary_embed(q, k, qw, kw, pos, sections), outs))


@TYPES
def test_the_python_path_gives_the_same(dtype, monkeypatch):
    t, h, hk, d, sections = 50, 3, 2, 64, (32,)
    q, k, gq, gk, qw, kw = _normal(7, dtype, (t, h, d), (t, hk, d), (t, h, d), (t, hk, d), (d,), (d,))
    pos = _positions(t, 1)
    outs, grads = _run(q, k, qw, kw, pos, sections, gq, gk)
    monkeypatch.setattr(_native, "binding", lambda: _native._NoBinding)
    o2, g2 = _run(q, k, qw, kw, pos, sections, gq, gk)
    assert all(torch.equal(x, y) for x, y in zip((*outs, *grads), (*o2, *g2)))
    _, g3 = _run(q, None, qw, None, pos, sections, gq, None)
    assert torch.equal(g3[0], grads[0]) and torch.equal(g3[2], grads[2])


@TYPES
def test_small_large_and_no_rows(dtype):
    """Rows of zeros, of tiny and of large numbers, a row that is not finite beside others, no tokens."""
    t, d, sections = 6, 64, (32,)
    (q,) = _normal(8, dtype, (t, 1, d))
    q[0], q[1], q[2] = 0, q[1] * 2.0 ** -60, q[2] * 2.0 ** 60
    (g, w) = _normal(9, dtype, (t, 1, d), (d,))
    pos = _positions(t, 1)
    outs, grads = _run(q, None, w, None, pos, sections, g, None)
    _check(outs, grads, q, None, w, None, pos, sections, g, None)
    assert not outs[0][0].any()
    bad = q.clone()
    bad[4, 0, 3] = float("inf")
    o2, g2 = _run(bad, None, w, None, pos, sections, g, None)
    keep = [0, 1, 2, 3, 5]
    assert torch.equal(o2[0][keep], outs[0][keep]) and torch.equal(g2[0][keep], grads[0][keep])
    assert torch.isnan(o2[0][4]).any()
    empty = torch.zeros(0, 2, d, dtype=dtype, device=_dev(), requires_grad=True)
    wl = w.detach().requires_grad_(True)
    out = norm_rotary_embed(empty, None, wl, None, pos[:0], sections)
    ge, gw = torch.autograd.grad(out, (empty, wl), torch.zeros_like(out))
    assert out.shape == empty.shape and ge.shape == empty.shape and not gw.any()


def test_refusals_on_a_gpu():
    q, k = _normal(10, torch.bfloat16, (4, 2, 64), (4, 1, 64))
    w, pos = torch.ones(64, device=_dev()), _positions(4, 1)
    ok = (q, k, w, w, pos, (32,))

    def swap(i, x):
        return (*ok[:i], x, *ok[i + 1:])

    for args, error, text in (
            (swap(0, q.half()), TypeError, "dtype"), (swap(1, k.float()), TypeError, "one type"), (swap(1, k[:3]), ValueError, "expected"),
            (swap(2, w.half()), TypeError, "q_weight"), (swap(2, w[:32]), ValueError, "q_weight"), (swap(3, w.cpu()), ValueError, "k_weight"),
            (swap(3, w.bfloat16()), TypeError, "one type"), (swap(1, None), ValueError, "without k"), (swap(4, pos.short()), TypeError, "positions"),
            (swap(4, pos[:3]), ValueError, "positions"), (swap(5, (33,)), ValueError, "pairs"), (swap(5, ()), ValueError, "sections")):
        with pytest.raises(error, match=text):
            norm_rotary_embed(*args)
    for options, text in ((dict(eps=0.0), "eps"), (dict(eps=float("nan")), "eps"), (dict(base=-1.0), "base")):
        with pytest.raises(ValueError, match=text):
            norm_rotary_embed(*ok, **options)
    out = norm_rotary_embed(q.detach().requires_grad_(True), k, w, w, pos, (32,))
    leaf = q.detach().requires_grad_(True)
    out = norm_rotary_embed(leaf, None, None, None, pos, (32,))
    (grad,) = torch.autograd.grad(out, leaf, torch.ones_like(out), create_graph=True)
    with pytest.raises(RuntimeError):
        grad.float().sum().backward()


@TYPES
def test_streams_and_graphs(dtype):
    """Two calls at once on two streams give the same bits each time; a captured step, replayed with other inputs and eager
    work between, gives the eager call's."""
    t, h, hk, d, sections = 300, 8, 2, 128, (16, 24, 24)
    sets = [_normal(11 + i, dtype, (t, h, d), (t, hk, d), (d,), (d,), (t, h, d), (t, hk, d)) for i in range(2)]
    pos = _positions(t, 3)

    def step(q, k, qw, kw, gq, gk):
        outs, grads = _run(q, k, qw, kw, pos, sections, gq, gk)
        return (*outs, *grads)

    want = [step(*s) for s in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(3):
        got = []
        for s, stream in zip(sets, streams):
            with torch.cuda.stream(stream):
                got.append(step(*s))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for x, y in zip(got, want) for a, b in zip(x, y))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(*sets[0])
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        outs = step(*sets[0])
    for i in range(3):
        sets[0][0].mul_(-1.5)
        pos.add_(i * 1000)
        eager = step(*sets[0])
        torch.cuda.synchronize()
        for x in outs:
            x.fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, eager)), i


@TYPES
def test_in_front_of_the_attention(dtype):
    """As it is used: queries and keys of one projection normed and turned, attended with capped scores in a window, and the
    gradients of the weights through both."""
    h, hk, d, off = 4, 2, 64, [0, 40, 95]
    (qkv, g, qw, kw) = _normal(13, dtype, (95, h + 2 * hk, d), (95, h, d), (d,), (d,))
    pos = torch.cat([torch.arange(40), torch.arange(55)])[:, None].to(torch.int32).to(_dev())
    offsets = torch.tensor(off, dtype=torch.int32, device=_dev())
    leaves = [x.detach().requires_grad_(True) for x in (qkv, qw, kw)]
    q, k = norm_rotary_embed(leaves[0][:, :h], leaves[0][:, h:h + hk], leaves[1], leaves[2], pos, (32,))
    out = packed_attention(q, k, leaves[0][:, h + hk:], offsets, cap=4.0, window=32)
    grads = torch.autograd.grad(out, leaves, g)
    shape, seqs = SA.Shape(cap=4.0, window=32), [(0, 40, 0, 40), (40, 55, 40, 55)]
    arrays = [_np(x) for x in (q, k, qkv[:, h + hk:], g)]
    bound = SA.bounds(*arrays, seqs, HALF_STEP[dtype], shape)
    _within(out, SA.attention(*arrays[:3], seqs, shape), bound[0], "out")
    gq, gk, gv = SA.attention_vjp(*arrays, seqs, shape)
    _within(grads[0][:, h + hk:], gv, bound[3], "grad_v")
    # the weights' gradients: those of the attention's own, whose errors pass through the norm's transpose
    p = pos.cpu().numpy()
    for i, (x, w, go, e, got) in enumerate(((qkv[:, :h], qw, gq, bound[1], grads[1]), (qkv[:, h:h + hk], kw, gk, bound[2], grads[2]))):
        _, dw = NR.backward(_np(x), _np(w), go, p, (32,), 1e-6)
        _, bw = NR.backward_bounds(_np(x), _np(w), np.abs(go) + e, p, (32,), 1e-6, HALF_STEP[dtype], HALF_STEP[dtype])
        through = (NR._pair_sum(e, (32,), False) * np.abs(_np(x)) * NR._root(_np(x), 1e-6)).sum((0, 1))
        _within(got, dw, bw + through * (1 + 2.0 ** -7), f"weight {i}")
