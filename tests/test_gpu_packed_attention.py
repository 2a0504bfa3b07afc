"""The attention over packed sequences (msda_packed_attention_fwd / _bwd through rfdetr_jax_amd.packed_attention)
on an MI355X, against the float64 oracle.

Tolerances are the oracle's ``bounds``: element by element, from half a step of the type for each weight
and result and 2^-24 for each term of an f32 sum.
"""

from __future__ import annotations

import sys

import numpy as np
import pytest
import torch

from oracle import packed_attention_ref as PA
from rfdetr_jax_amd import packed_attention, packed_attention_backward, packed_attention_forward, rotary_embed

pytestmark = pytest.mark.gpu
HALF_STEP = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}
TYPES = pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])


def _note(msg):
    sys.stderr.write(f"[gpu] {msg}\n")
    sys.stderr.flush()


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
    assert got.shape == want.shape, what
    assert np.isfinite(got).all(), f"{what}: not finite"
    over = np.abs(got - want) - bound
    at = np.unravel_index(np.argmax(over), over.shape)
    assert over[at] <= 0, f"{what}: off by {abs(got[at] - want[at]):.3e} at {at}, {bound[at]:.3e} allowed"


def _compare(q, k, v, g, got, seqs, causal, scale=None):
    arrays = [_np(x) for x in (q, k, v, g)]
    want = [PA.attention(*arrays[:3], seqs, causal, scale), *PA.attention_vjp(*arrays, seqs, causal, scale)]
    bound = PA.bounds(*arrays, seqs, HALF_STEP[q.dtype], causal, scale)
    for name, x, w, b in zip(("out", "grad_q", "grad_k", "grad_v"), got, want, bound):
        if x is not None:
            _within(x, w, b, name)


def _run(q, k, v, g, offsets, key_offsets=None, key_lengths=None, causal=True, scale=None):
    leaves = [x.detach().requires_grad_(True) for x in (q, k, v)]
    out = packed_attention(*leaves, offsets, key_offsets, key_lengths, causal, scale)
    assert out.shape == q.shape and out.dtype == q.dtype
    return (out, *torch.autograd.grad(out, leaves, g))


#      lengths, keys, heads, key heads, head dim
SHAPES = {
    "one_token": ([1], [1], 1, 1, 32),
    "ragged": ([5, 64, 1, 130, 33, 0, 63], None, 4, 2, 64),
    "odd_group": ([43, 7, 90], None, 6, 2, 128),       # rows of a tile in groups of 3
    "one_key_head": ([100, 29], None, 8, 1, 64),
    "dim8": ([70, 3], None, 2, 2, 8),
    "dim40": ([65, 31], None, 3, 1, 40),
    "dim96": ([129, 40], None, 2, 1, 96),
    "dim120": ([50, 66], None, 2, 2, 120),
    "more_keys": ([3, 70, 0, 20], [200, 70, 5, 65], 4, 2, 64),
    "fewer_keys": ([40, 9, 130], [10, 0, 127], 4, 2, 32),  # rows that see no key
    "long": ([700, 1], None, 2, 1, 128),
}


@TYPES
@pytest.mark.parametrize("causal", [False, True], ids=["all", "causal"])
@pytest.mark.parametrize("name", sorted(SHAPES))
def test_against_oracle(name, causal, dtype):
    lengths, keys, h, hk, d = SHAPES[name]
    keys = lengths if keys is None else keys
    _note(f"packed attention {name} causal={causal} {dtype}")
    off, koff = np.cumsum([0, *lengths]), np.cumsum([0, *keys])
    q, k, v, g = _normal(5, dtype, (off[-1], h, d), (koff[-1], hk, d), (koff[-1], hk, d), (off[-1], h, d))
    got = _run(q, k, v, g, _int(off), _int(koff), causal=causal)
    _compare(q, k, v, g, got, PA.sequences(off, koff), causal)


@TYPES
def test_large_scores_and_scale(dtype):
    """Scores that rise and fall by hundreds along the keys: the running reference score moves and rows are dominated by
    one key."""
    off = [0, 300, 333]
    q, k, v, g = _normal(6, dtype, (333, 2, 64), (333, 1, 64), (333, 1, 64), (333, 2, 64))
    ramp = torch.linspace(0.2, 6.0, 333, device=_dev())[:, None, None].to(dtype)
    for kk in (k * ramp, k * ramp.flip(0)):
        for scale in (None, 0.7):
            got = _run(q, kk, v, g, _int(off), scale=scale)
            _compare(q, kk, v, g, got, PA.sequences(off), True, scale)


@TYPES
def test_rows_outside_the_sequences(dtype):
    """Rows before the first sequence, behind the last, and of a cache behind its keys: they hold NaN, take no part and
    come out as zeros."""
    off, koff, lengths = [3, 60, 60, 190], [7, 90, 140, 300], [57, 20, 130]
    q, k, v, g = _normal(7, dtype, (200, 4, 64), (320, 2, 64), (320, 2, 64), (200, 4, 64))
    seqs = PA.sequences(off, koff, lengths)
    for x in (q, g):
        x[:3] = x[190:] = float("nan")
    outside = torch.ones(320, dtype=torch.bool, device=_dev())
    for _, _, k0, m in seqs:
        outside[k0:k0 + m] = False
    k[outside] = v[outside] = float("nan")
    got = _run(q, k, v, g, _int(off), _int(koff), _int(lengths))
    for x in (got[0], got[1]):
        assert not x[:3].any() and not x[190:].any()
    for x in got[2:]:
        assert not x[outside].any()
    clean = [torch.nan_to_num(x) for x in (q, k, v, g)]
    _compare(*clean, got, seqs, True)


@TYPES
def test_slices_of_a_projection_and_other_strides(dtype):
    """q, k and v as slices of one projection's rows; head-major tensors; rows off their 16-byte boundaries (copied);
    channels that are not contiguous; a key head for all rows by stride 0; a cotangent by stride 0."""
    off = [0, 50, 131]
    h, hk, d, seqs = 4, 2, 64, PA.sequences(off)
    (qkv,) = _normal(8, dtype, (131, (h + 2 * hk) * d + 8))
    flat = qkv[:, :-8].unflatten(1, (h + 2 * hk, d))
    parts = [flat[:, :h], flat[:, h:h + hk], flat[:, h + hk:]]
    (g,) = _normal(9, dtype, (131, h, d))
    want = _run(*(x.contiguous() for x in parts), g, _int(off))
    _compare(*parts, g, want, seqs, True)
    head_major = [x.transpose(0, 1).contiguous().transpose(0, 1) for x in parts]
    shifted = [torch.empty(x.numel() + 1, dtype=dtype, device=_dev())[1:].view(x.shape).copy_(x) for x in parts]
    channels = [x.transpose(1, 2).contiguous().transpose(1, 2) for x in parts]
    for other in (parts, head_major, shifted, channels):
        got = _run(*other, g, _int(off))
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    one = [parts[0], parts[1][:1].expand(131, hk, d), parts[2]]
    got = _run(*one, g, _int(off))
    _compare(*one, g, got, seqs, True)
    ones = torch.ones((), dtype=dtype, device=_dev()).expand(131, h, d)
    _compare(*parts, ones, _run(*parts, ones, _int(off)), seqs, True)


@TYPES
@pytest.mark.parametrize("new", [1, 7], ids=["one_token", "chunk"])
@pytest.mark.parametrize("heads", [(8, 1), (4, 4), (16, 2)], ids=["8to1", "4to4", "16to2"])
def test_tokens_over_a_cache(heads, new, dtype):
    """Few new tokens over caches of different fill (one key, a tile less one, many), whose keys are split over
    workgroups; unfilled rows hold NaN. A sequence without new tokens and one without keys are among them."""
    h, hk = heads
    room, fill, d = 2500, [2500, 1, 63, 0, 1999, 64], 128
    lengths = [min(new, max(m, 1)) for m in fill]
    lengths[4] = 0
    off, koff = np.cumsum([0, *lengths]), np.arange(len(fill) + 1) * room
    q, k, v = _normal(10, dtype, (off[-1], h, d), (koff[-1], hk, d), (koff[-1], hk, d))
    for i, m in enumerate(fill):
        k[koff[i] + m:koff[i + 1]] = v[koff[i] + m:koff[i + 1]] = float("nan")
    out = packed_attention(q, k, v, _int(off), _int(koff), _int(fill))
    seqs = PA.sequences(off, koff, fill)
    _compare(q, torch.nan_to_num(k), torch.nan_to_num(v), torch.zeros_like(q), (out,), seqs, True)
    out2, stats = packed_attention_forward(q, k, v, _int(off), _int(koff), _int(fill))
    assert torch.equal(out, out2)
    (g,) = _normal(11, dtype, q.shape)
    grads = packed_attention_backward(q, k, v, out2, stats, g, _int(off), _int(koff), _int(fill))
    _compare(q, torch.nan_to_num(k), torch.nan_to_num(v), g, (out2, *grads), seqs, True)


@TYPES
def test_gradients_wanted_one_by_one(dtype):
    off = [0, 77, 140]
    q, k, v, g = _normal(12, dtype, (140, 4, 64), (140, 2, 64), (140, 2, 64), (140, 4, 64))
    out, stats = packed_attention_forward(q, k, v, _int(off))
    want = packed_attention_backward(q, k, v, out, stats, g, _int(off))
    for i in range(3):
        needs = [j == i for j in range(3)]
        got = packed_attention_backward(q, k, v, out, stats, g, _int(off), needs=needs)
        assert [x is not None for x in got] == needs and torch.equal(got[i], want[i])
        leaves = [x.detach().requires_grad_(j == i) for j, x in enumerate((q, k, v))]
        (grad,) = torch.autograd.grad(packed_attention(*leaves, _int(off)), [leaves[i]], g)
        assert torch.equal(grad, want[i])
    with torch.no_grad():
        assert torch.equal(packed_attention(q, k, v, _int(off)), out)


def test_empty_calls():
    d = _dev()
    for t, s, n in ((0, 0, 0), (0, 5, 1), (4, 0, 1), (4, 5, 0), (4, 5, 2)):
        q = torch.randn(t, 2, 32, device=d, requires_grad=True)
        k, v = (torch.randn(s, 1, 32, device=d, requires_grad=True) for _ in range(2))
        off, koff = torch.zeros(n + 1, dtype=torch.int32, device=d), torch.zeros(n + 1, dtype=torch.int32, device=d)
        out = packed_attention(q, k, v, off, koff)
        grads = torch.autograd.grad(out, (q, k, v), torch.ones_like(out))
        assert not out.any() and not any(x.any() for x in grads)


def test_offsets_that_do_not_rise_stay_in_bounds():
    """Falling, negative and too large offsets and lengths are clamped: the call ends and a following right call is right."""
    q, k, v, g = _normal(13, torch.float32, (150, 4, 32), (300, 2, 32), (300, 2, 32), (150, 4, 32))
    for off, koff, lengths in (([0, 150, 20, 150], [0, 300, 10, 300], None), ([-5, 40, 1000, 2000], [-9, 100, 400, 9000], [900, -3, 50]),
                               ([150, 0, 0, 0], [300, 0, 0, 0], [3, 3, 3])):
        got = _run(q, k, v, g, _int(off), _int(koff), None if lengths is None else _int(lengths))
        assert [x.shape for x in got] == [q.shape, q.shape, k.shape, v.shape]
    off, koff = [0, 100, 150], [0, 200, 300]
    _compare(q, k, v, g, _run(q, k, v, g, _int(off), _int(koff)), PA.sequences(off, koff), True)


@TYPES
def test_the_same_bits_each_time_and_beside_other_work(dtype):
    """Two calls at once on two streams, and again: the same bits."""
    off = _int([0, 200, 513, 600])
    a = _normal(14, dtype, (600, 8, 64), (600, 2, 64), (600, 2, 64), (600, 8, 64))
    b = _normal(15, dtype, (600, 8, 64), (600, 2, 64), (600, 2, 64), (600, 8, 64))
    want = [_run(*x, off) for x in (a, b)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(3):
        got = []
        for x, s in zip((a, b), streams):
            with torch.cuda.stream(s):
                got.append(_run(*x, off))
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for x, y in zip(got, want) for p, q in zip(x, y))


@TYPES
def test_in_a_graph_with_other_lengths(dtype):
    """One captured forward and backward, and a captured call with split keys, replayed with other lengths, offsets and
    inputs and other eager work between: each replay gives the eager call's bits."""
    q, k, v, g = _normal(16, dtype, (300, 4, 64), (300, 2, 64), (300, 2, 64), (300, 4, 64))
    off = _int([0, 100, 300])
    cq, ck, cv = _normal(17, dtype, (2, 4, 64), (4000, 2, 64), (4000, 2, 64))
    coff, ckoff, fill = _int([0, 1, 2]), _int([0, 2000, 4000]), _int([2000, 5])

    def work():
        out, stats = packed_attention_forward(q, k, v, off)
        return (out, *packed_attention_backward(q, k, v, out, stats, g, off), packed_attention(cq, ck, cv, coff, ckoff, fill))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        work()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        outs = work()
    for lengths, filled in (([0, 100, 300], [2000, 5]), ([0, 0, 177], [1, 1999]), ([20, 21, 290], [0, 700])):
        off.copy_(_int(lengths))
        fill.copy_(_int(filled))
        q.mul_(-0.5)
        eager = work()
        torch.cuda.synchronize()
        for x in outs:
            x.fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, eager)), (lengths, filled)


@TYPES
def test_rotary_prompt_and_tokens(dtype):
    """As they are used together: a step of training on packed sequences with positions on three axes, and the same
    sequences again token by token over a cache, whose last tokens agree with the prompt's within the bounds."""
    h, hk, d, lengths, room = 4, 2, 64, [37, 70], 128
    off = np.cumsum([0, *lengths])
    (qkv,) = _normal(18, dtype, (off[-1], h + 2 * hk, d))
    (g,) = _normal(19, dtype, (off[-1], h, d))
    pos = torch.stack([torch.cat([torch.arange(n) for n in lengths])] * 3, 1).to(torch.int32).to(_dev())
    leaf = qkv.detach().requires_grad_(True)
    q, k = rotary_embed(leaf[:, :h], leaf[:, h:h + hk], pos, (8, 12, 12), shared_frequencies=True)
    out = packed_attention(q, k, leaf[:, h + hk:], _int(off))
    (grad,) = torch.autograd.grad(out, leaf, g)
    seqs = PA.sequences(off)
    v = qkv[:, h + hk:]
    arrays = [_np(x) for x in (q, k, v, g)]
    bound = PA.bounds(*arrays, seqs, HALF_STEP[dtype])
    _within(out, PA.attention(*arrays[:3], seqs), bound[0], "out")
    _within(grad[:, h + hk:], PA.attention_vjp(*arrays, seqs)[2], bound[3], "grad_v")
    # the gradient of the unrotated keys: a rotation mixes two channels' errors, and rounds once
    from oracle import rotary_ref as RO

    for at, i in ((slice(0, h), 1), (slice(h, h + hk), 2)):
        want = RO.rotate(PA.attention_vjp(*arrays, seqs)[i - 1], pos.cpu().numpy(), (8, 12, 12), shared=True, sign=-1.0)
        e = bound[i]
        both = np.concatenate([e[..., :32] + e[..., 32:]] * 2, -1)
        _within(grad[:, at], want, both + (HALF_STEP[dtype] + 2.0 ** -20) * (np.abs(want) + both), "grad of the projection")
    # token by token
    cache = [torch.full((len(lengths) * room, hk, d), float("nan"), dtype=dtype, device=_dev()) for _ in range(2)]
    starts = _int(np.arange(len(lengths) + 1) * room)
    for i, n in enumerate(lengths):
        cache[0][i * room:i * room + n - 1], cache[1][i * room:i * room + n - 1] = k.detach()[off[i]:off[i + 1] - 1], v[off[i]:off[i + 1] - 1]
    last = torch.tensor(off[1:] - 1, device=_dev())
    nq, nk = rotary_embed(qkv[last, :h], qkv[last, h:h + hk], pos[last], (8, 12, 12), shared_frequencies=True)
    assert torch.equal(nq, q[last]) and torch.equal(nk, k[last])
    rows = torch.tensor([i * room + n - 1 for i, n in enumerate(lengths)], device=_dev())
    cache[0][rows], cache[1][rows] = nk, v[last]
    got = packed_attention(nq, *cache, _int([0, 1, 2]), starts, _int(lengths))
    at = last.cpu().numpy()
    _within(got, PA.attention(*arrays[:3], seqs)[at], bound[0][at], "token by token")


#        queries, keys, heads, key heads, head dim; the key and the query that are spoilt
SPOILT = {
    "square": (150, 150, 4, 2, 64, 100, 20),
    "tile_edge": (192, 192, 1, 1, 32, 127, 64),
    "one_key_head": (200, 230, 8, 1, 128, 200, 11),
    "odd_group": (90, 300, 6, 2, 40, 280, 3),
    "over_a_cache": (9, 2100, 4, 1, 128, 2095, 2),  # the keys are split
    "last": (65, 65, 2, 2, 96, 64, 64),
}


@TYPES
@pytest.mark.parametrize("value", [float("nan"), float("inf"), -float("inf")], ids=["nan", "inf", "minus_inf"])
@pytest.mark.parametrize("name", sorted(SPOILT))
def test_unseen_pairs_take_no_part_whatever_they_hold(name, value, dtype):
    """Rows that do not see a value that is no finite number keep their results to the bit, those that see it do not."""
    n, m, h, hk, d, key, query = SPOILT[name]
    _note(f"packed attention unseen {name} {value} {dtype}")
    shift = m - n
    off, koff = [0, n, n + 30], [0, m, m + 30]
    q, k, v, g = _normal(21, dtype, (n + 30, h, d), (m + 30, hk, d), (m + 30, hk, d), (n + 30, h, d))
    args = (_int(off), _int(koff))
    clean = _run(q, k, v, g, *args)
    _compare(q, k, v, g, clean, PA.sequences(off, koff), True)
    sees = max(key - shift, 0)  # the first query that sees the key

    bad_v = v.clone()
    bad_v[key, :, 5] = value
    out, gq, gk, gv = _run(q, k, bad_v, g, *args)
    others = [c for c in range(d) if c != 5]
    assert torch.equal(out[:sees], clean[0][:sees]) and torch.equal(out[n:], clean[0][n:])
    assert torch.equal(out[sees:n, :, others], clean[0][sees:n, :, others])
    assert not torch.isfinite(out[sees:n, :, 5]).any()
    assert torch.equal(gq[:sees], clean[1][:sees]) and torch.equal(gq[n:], clean[1][n:])
    assert torch.equal(gk[m:], clean[2][m:]) and torch.equal(gv[m:], clean[3][m:])
    assert torch.isnan(gq[sees:n]).any()

    bad_k = k.clone()
    bad_k[key, :, 5] = value
    out, gq, gk, gv = _run(q, bad_k, v, g, *args)
    for x, c, first, last in ((out, clean[0], sees, n), (gq, clean[1], sees, n), (gk, clean[2], m, m), (gv, clean[3], m, m)):
        if first < last:
            assert torch.equal(x[:first], c[:first])
        assert torch.equal(x[last:], c[last:])
    assert torch.isnan(gq[sees:n]).any()

    unseen = query + shift + 1  # the first key that the query does not see
    for which in range(2):
        q2, g2 = q.clone(), g.clone()
        (q2, g2)[which][query, :, 7] = value
        out, gq, gk, gv = _run(q2, k, v, g2, *args)
        for x, c in ((out, clean[0]), (gq, clean[1])):
            assert torch.equal(x[:query], c[:query]) and torch.equal(x[query + 1:], c[query + 1:])
        for x, c in ((gk, clean[2]), (gv, clean[3])):
            assert torch.equal(x[unseen:], c[unseen:])
        assert not torch.isfinite(gk[:unseen]).all() and not torch.isfinite(gq[query]).all()


@TYPES
@pytest.mark.parametrize("causal", [False, True], ids=["all", "causal"])
def test_keys_behind_the_length_get_zeros_where_queries_are_not_finite(causal, dtype):
    off, koff, lengths = [0, 40], [0, 100], [70]
    q, k, v, g = _normal(22, dtype, (40, 2, 128), (100, 2, 128), (100, 2, 128), (40, 2, 128))
    for which in range(2):
        q2, g2 = q.clone(), g.clone()
        (q2, g2)[which][3] = float("nan")
        _, _, gk, gv = _run(q2, k, v, g2, _int(off), _int(koff), _int(lengths), causal=causal)
        assert not gk[70:].any() and not gv[70:].any()
        assert torch.isnan(gk[:33]).all()


#      lengths, keys, heads, key heads, head dim
WIDE = {
    "thousands": ([int(i * 7919 % 4) for i in range(5000)], None, 2, 1, 8),
    "sixty_four_to_a_head": ([40, 3], [50, 3], 64, 1, 64),
    "thirty_three_to_a_head": ([30, 66], None, 66, 2, 32),
    "one_token_in_many": ([0] * 100 + [1] + [0] * 100, [0] * 100 + [333] + [0] * 100, 64, 2, 128),
    "long_keys": ([130, 2], [4000, 3000], 2, 1, 128),
}


@TYPES
@pytest.mark.parametrize("name", sorted(WIDE))
def test_many_sequences_wide_groups_and_long_keys(name, dtype):
    lengths, keys, h, hk, d = WIDE[name]
    keys = lengths if keys is None else keys
    _note(f"packed attention {name} {dtype}")
    off, koff = np.cumsum([0, *lengths]), np.cumsum([0, *keys])
    q, k, v, g = _normal(23, dtype, (off[-1], h, d), (koff[-1], hk, d), (koff[-1], hk, d), (off[-1], h, d))
    for causal in (False, True):
        got = _run(q, k, v, g, _int(off), _int(koff), causal=causal)
        _compare(q, k, v, g, got, PA.sequences(off, koff), causal)


@TYPES
def test_rows_far_apart(dtype):
    """A cache whose rows lie beyond 2^31 elements, and heads in front of the rows (head-major), without a copy."""
    h, hk, d, stride, fill = 4, 2, 64, 1 << 14, [90, 300]
    first = [(1 << 31) // stride + 5, (1 << 31) // stride + 400]
    rows = first[1] + 400
    store = torch.empty(rows * stride, dtype=dtype, device=_dev())
    k, v = (store.view(rows, stride)[:, at:at + hk * d].unflatten(1, (hk, d)) for at in (0, hk * d))
    koff, off = [*first, rows], [0, 90, 95]
    small = _normal(24, dtype, (rows - first[0], hk, d), (rows - first[0], hk, d), (95, h, d), (95, h, d))
    k[first[0]:], v[first[0]:] = small[:2]
    q, g = small[2:]
    out, saved = packed_attention_forward(q, k, v, _int(off), _int(koff), _int(fill))
    grads = packed_attention_backward(q, k, v, out, saved, g, _int(off), _int(koff), _int(fill))
    near = [0, first[1] - first[0], rows - first[0]]
    tail = (out, grads[0], *(x[first[0]:] for x in grads[1:]))
    assert not any(x[:first[0]].any() for x in grads[1:])
    _compare(q, *small[:2], g, tail, PA.sequences(off, near, fill), True)
    major = store.view(-1)[:2 * hk * (1 << 29)].view(2, hk, -1, d)  # a head lies 2^29 elements behind the one before
    kk, vv = (x.transpose(0, 1)[-400:] for x in major)
    kk.copy_(small[0][:400]), vv.copy_(small[1][:400])
    got = packed_attention_forward(q, kk, vv, _int(off), _int([0, 90, 400]), _int([90, 300]))[0]
    want = packed_attention_forward(q, small[0][:400], small[1][:400], _int(off), _int([0, 90, 400]), _int([90, 300]))[0]
    assert torch.equal(got, want)


@TYPES
def test_both_ways_in_give_the_same_bits(dtype):
    """The C++ function and the Python one, which takes what the first does not; 64-bit offsets."""
    from rfdetr_jax_amd.packed_attention import _PackedAttention

    off, koff, lengths = [0, 33, 150], [0, 100, 260], [70, 160]
    q, k, v, g = _normal(25, dtype, (150, 4, 64), (260, 2, 64), (260, 2, 64), (150, 4, 64))
    args = (_int(off), _int(koff), _int(lengths))
    want = _run(q, k, v, g, *args, scale=0.3)
    leaves = [x.detach().requires_grad_(True) for x in (q, k, v)]
    out = _PackedAttention.apply(*leaves, *args, True, 0.3)
    got = (out, *torch.autograd.grad(out, leaves, g))
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    got = _run(q, k, v, g, *(x.long() for x in args), scale=0.3)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_gradients_are_not_differentiable_again():
    from rfdetr_jax_amd.packed_attention import _PackedAttention

    q, k, v, g = (x.requires_grad_(True) for x in _normal(26, torch.float32, (10, 2, 32), (10, 1, 32), (10, 1, 32), (10, 2, 32)))
    for call in (packed_attention, lambda *a: _PackedAttention.apply(*a, None, None, True, None)):
        (grad,) = torch.autograd.grad(call(q, k, v, _int([0, 10])), [q], g, create_graph=True)
        with pytest.raises(RuntimeError, match="differentiate"):
            torch.autograd.grad(grad.sum(), [q])


def test_front_end_refusals():
    d = _dev()
    q, k, off = torch.zeros(6, 4, 32, device=d), torch.zeros(6, 2, 32, device=d), _int([0, 6])
    for args, error, text in (
            ((q.double(), k.double(), k.double(), off), TypeError, "not supported"), ((q, k.bfloat16(), k, off), TypeError, "one type"),
            ((q[0], k, k, off), ValueError, "rows, heads, D"), ((q, k, k[:5], off), ValueError, "expected"), ((q, k[..., :16], k[..., :16], off), ValueError, "expected"),
            ((q[:, :3], k, k, off), ValueError, "divide"), ((q, k[:, :0], k[:, :0], off), ValueError, "divide"), ((q[:, :0], k, k, off), ValueError, "divide"),
            ((q.repeat(1, 33, 1), k, k, off), ValueError, "share"), ((q[..., :12], k[..., :12], k[..., :12], off), ValueError, "head_dim"),
            ((q.repeat(1, 1, 5), k.repeat(1, 1, 5), k.repeat(1, 1, 5), off), ValueError, "head_dim"), ((q[..., :0], k[..., :0], k[..., :0], off), ValueError, "head_dim"),
            ((q, k, k, off.float()), TypeError, "int32"), ((q, k, k, off[None]), ValueError, "offsets"), ((q, k, k, off[:0]), ValueError, "offsets"),
            ((q, k, k, off, _int([0, 3, 6])), ValueError, "key_offsets"), ((q, k, k, off, None, _int([1, 2])), ValueError, "key_lengths"),
            ((q, k, k, off.cpu()), ValueError, "cpu"), ((q, k, k, off, None, _int([6]).cpu()), ValueError, "cpu"), ((q, k.cpu(), k, off), RuntimeError, "no CPU path"),
            ((q, k, k, off, None, None, True, 0.0), ValueError, "scale"), ((q, k, k, off, None, None, True, float("nan")), ValueError, "scale"),
            ((q, k, k, off, None, None, True, 1e-30), ValueError, "scale")):
        with pytest.raises(error, match=text):
            packed_attention(*args)
        with pytest.raises(error, match=text):
            packed_attention_forward(*args)
    out, saved = packed_attention_forward(q, k, k, off)
    for bad in ((out[:5], saved, q), (out, (saved[0][:, :2], None), q), (out, saved, q[:, :2]), (out, saved, q.cpu())):
        with pytest.raises(ValueError):
            packed_attention_backward(q, k, k, *bad, off)


@TYPES
@pytest.mark.parametrize("count", [61, 62, 63, 126, 1021, 1022, 1023])
def test_numbers_of_sequences_where_the_search_changes(count, dtype):
    """64 segments of rows fit a wave, 1,024 are counted, more are searched; equal lengths, none and longer ones among them."""
    lengths = [i * 7 % 5 if i % 11 else 0 for i in range(count)]
    lengths[count // 2] = 140
    off = np.cumsum([0, *lengths])
    q, k, v, g = _normal(27, dtype, (off[-1], 2, 32), (off[-1], 1, 32), (off[-1], 1, 32), (off[-1], 2, 32))
    got = _run(q, k, v, g, _int(off))
    _compare(q, k, v, g, got, PA.sequences(off), True)
    fill = [n + 100 + i % 37 for i, n in enumerate(lengths)]  # few rows, split keys
    koff = np.cumsum([0, *(m + 3 for m in fill)])
    k, v = _normal(28, dtype, (koff[-1], 1, 32), (koff[-1], 1, 32))
    out = packed_attention(q, k, v, _int(off), _int(koff), _int(fill))
    _compare(q, k, v, torch.zeros_like(q), (out,), PA.sequences(off, koff, fill), True)


#        queries, keys, heads, key heads, head dim, causal; the key that is spoilt
SEEN = {
    "short": (40, 40, 2, 1, 64, False, 11),
    "one_token": (1, 63, 8, 2, 128, True, 20),
    "one_key": (5, 1, 2, 2, 32, False, 0),
    "two_tiles": (150, 63, 4, 4, 32, False, 62),
    "causal": (63, 63, 4, 2, 64, True, 0),
    "chunk": (7, 50, 4, 1, 40, True, 30),
    "short_rows_of_a_long_prompt": (200, 200, 2, 2, 96, True, 5),
    "whole_tile": (70, 64, 2, 1, 128, False, 40),
    "long": (30, 300, 4, 2, 64, False, 299),
    "token_over_a_cache": (1, 2000, 8, 1, 128, True, 1234),  # the keys are split
    "chunk_over_a_cache": (7, 500, 4, 1, 64, True, 498),
    "many_rows": (40, 500, 4, 1, 64, True, 300),
}


@TYPES
@pytest.mark.parametrize("name", sorted(SEEN))
def test_infinities_of_seen_values_come_out_as_they_are(name, dtype):
    """Every weight of these rows is above 0, so an infinity in a channel of a value gives that infinity where it is seen,
    both signs together and NaN give NaN; the other channels, and the rows that do not see it, keep their bits."""
    n, m, h, hk, d, causal, key = SEEN[name]
    _note(f"packed attention seen infinities {name} {dtype}")
    q, k, v = _normal(29, dtype, (n + 9, h, d), (m + 9, hk, d), (m + 9, hk, d))
    args = (_int([0, n, n + 9]), _int([0, m, m + 9]), None, causal)
    clean = packed_attention(q, k, v, *args)
    assert torch.isfinite(clean).all()
    sees = max(key - (m - n), 0) if causal else 0
    bad = v.clone()
    bad[key, :, 3], bad[key, :, 4], bad[key, :, d - 1] = float("inf"), -float("inf"), float("nan")
    wrong = [3, 4, d - 1]
    if m > 1:  # a second key, seen by fewer or more rows: both signs in one channel
        other = key - 1 if key else 1
        bad[key, :, 6], bad[other, :, 6] = float("inf"), -float("inf")
        wrong.append(6)
    out = packed_attention(q, k, bad, *args)
    last = max(key, other if m > 1 else 0)
    first = sees if m == 1 or not causal else min(sees, max(other - (m - n), 0))
    both = sees if m == 1 or not causal else max(last - (m - n), 0)
    rest = [c for c in range(d) if c not in wrong]
    assert torch.equal(out[:first], clean[:first]) and torch.equal(out[n:], clean[n:])
    assert torch.equal(out[:n, :, rest], clean[:n, :, rest])
    for at, value in ((3, float("inf")), (4, -float("inf"))):
        assert torch.equal(out[sees:n, :, at], torch.full_like(out[sees:n, :, at], value))
        assert torch.equal(out[:sees, :, at], clean[:sees, :, at])
    assert torch.isnan(out[sees:n, :, d - 1]).all()
    if m > 1:
        assert torch.isnan(out[both:n, :, 6]).all()


@TYPES
def test_backward_leaves_what_the_forward_saved(dtype):
    """The statistics and the rest are read alone: one forward serves several cotangents, on two streams at once, too."""
    off = _int([0, 300, 513, 600])
    q, k, v, g, g2 = _normal(30, dtype, (600, 8, 64), (600, 2, 64), (600, 2, 64), (600, 8, 64), (600, 8, 64))
    out, (stats, rest) = packed_attention_forward(q, k, v, off)
    stats[..., 2:] = 7.0  # (no part of the statistics)
    before = [None if x is None else x.clone() for x in (out, stats, rest)]
    want = [packed_attention_backward(q, k, v, out, (stats, rest), x, off) for x in (g, g2)]
    for x, y in zip((out, stats, rest), before):
        assert (x is None and y is None) or torch.equal(x, y)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(5):
        got = []
        for x, s in zip((g, g2), streams):
            with torch.cuda.stream(s):
                got.append(packed_attention_backward(q, k, v, out, (stats, rest), x, off))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for x, y in zip(got, want) for a, b in zip(x, y))
    # the autograd function: one graph, two cotangents
    leaves = [x.detach().requires_grad_(True) for x in (q, k, v)]
    out = packed_attention(*leaves, off)
    got = [torch.autograd.grad(out, leaves, x, retain_graph=True) for x in (g, g2, g)]
    assert all(torch.equal(a, b) for x, y in zip(got, (*want, want[0])) for a, b in zip(x, y))


@pytest.mark.parametrize("causal", [False, True], ids=["all", "causal"])
@pytest.mark.parametrize("late", [False, True], ids=["level", "late_maximum"])
def test_short_bf16_rows_keep_what_the_weights_rounding_left(late, causal):
    """Rows of fewer than 64 keys. A weight is the sum of two bf16 numbers, off by half a step of half a step (2^-16 of it);
    the result rounds once. With a late maximum the last keys outweigh the first 32, whose values are as much
    larger, by 2^11: the rest of those weights is scaled with them."""
    n, d = 60, 64
    q, k, v = _normal(31, torch.bfloat16, (n, 4, d), (n, 2, d), (n, 2, d))
    if late:
        q[..., 0], k[..., 0] = 8, 0
        k[32:, :, 0] = 8  # 8 of a score: 11.5 of its log2
        v[:32] *= 2.0 ** 11
    out = packed_attention(q, k, v, _int([0, n]), causal=causal)
    arrays, seqs = [_np(x) for x in (q, k, v)], PA.sequences([0, n])
    want = PA.attention(*arrays, seqs, causal)
    bound = PA.bounds(*arrays, np.zeros_like(arrays[0]), seqs, 2.0 ** -16, causal)[0]
    _within(out, want, (1 + 2.0 ** -8) * bound + 2.0 ** -8 * np.abs(want), "out")


#      lengths, keys, heads, key heads, head dim: the numbers of parts of a sequence's tiles grow
GROWING = {
    "prompts": ([1500, 400, 33], None, 8, 8, 64),
    "group_of_three": ([1100, 700], None, 6, 2, 32),
    "fewer_keys": ([1500, 900], [1100, 900], 4, 4, 40),  # tiles without keys in front
    "more_keys": ([900, 640, 2], [1700, 700, 500], 2, 2, 128),
    "seventy_tiles": ([4250], None, 2, 1, 32),
    "seventy_sequences": ([300 + i * 397 % 500 for i in range(70)], None, 1, 1, 32),
}


@TYPES
@pytest.mark.parametrize("name", sorted(GROWING))
def test_tiles_with_more_parts_the_more_keys_they_see(name, dtype):
    from rfdetr_jax_amd import _native

    lengths, keys, h, hk, d = GROWING[name]
    keys = lengths if keys is None else keys
    _note(f"packed attention parts {name} {dtype}")
    off, koff = np.cumsum([0, *lengths]), np.cumsum([0, *keys])
    code = _native.DTYPE_BF16 if dtype == torch.bfloat16 else _native.DTYPE_F32
    assert _native.lib().msda_packed_attention_fwd_workspace_size(code, len(lengths), off[-1], koff[-1], h, hk, d) > 0
    q, k, v, g = _normal(32, dtype, (off[-1], h, d), (koff[-1], hk, d), (koff[-1], hk, d), (off[-1], h, d))
    got = _run(q, k, v, g, _int(off), _int(koff))
    _compare(q, k, v, g, got, PA.sequences(off, koff), True)


def test_offsets_that_fall_and_rise_over_many_rows_stay_in_bounds():
    """A thousand sequences over the same 25 million rows of 64 heads: the sum of their tiles passes 32 bits. The call ends, and
    a right one behind it is right."""
    rows = 25_000_000
    q = torch.empty(rows, 64, 8, dtype=torch.bfloat16, device=_dev())
    k = torch.zeros(1, 1, 8, dtype=torch.bfloat16, device=_dev())
    off = _int([0 if i % 2 == 0 else rows for i in range(1001)])
    out = packed_attention(q, k, k, off, torch.zeros_like(off), causal=False)
    torch.cuda.synchronize()
    assert out.shape == q.shape
    del q, out
    torch.cuda.empty_cache()
    off = [0, 100, 150]
    q, k, v, g = _normal(33, torch.bfloat16, (150, 4, 32), (150, 2, 32), (150, 2, 32), (150, 4, 32))
    _compare(q, k, v, g, _run(q, k, v, g, _int(off)), PA.sequences(off), True)


@pytest.mark.parametrize("d", [40, 64, 128])
def test_new_bf16_tokens_keep_what_the_weights_rounding_left(d):
    """Sequences of at most 32 rows over caches of any length, split or not: the two bf16 numbers of a weight, as for short
    rows."""
    lengths, keys = [1, 3, 4, 2], [2000, 700, 100, 1300]
    off, koff = np.cumsum([0, *lengths]), np.cumsum([0, *keys])
    q, k, v = _normal(34, torch.bfloat16, (off[-1], 8, d), (koff[-1], 1, d), (koff[-1], 1, d))
    seqs = PA.sequences(off, koff)
    for factor in (1, 4):  # sums of many keys, and rows that a few of them make
        out = packed_attention(q * factor, k, v, _int(off), _int(koff))
        arrays = [_np(x) for x in (q * factor, k, v)]
        want = PA.attention(*arrays, seqs)
        bound = PA.bounds(*arrays, np.zeros_like(arrays[0]), seqs, 2.0 ** -16)[0]
        _within(out, want, (1 + 2.0 ** -8) * bound + 2.0 ** -8 * np.abs(want), "out")


@TYPES
def test_c_entry_that_keeps_its_numbers_in_the_statistics(dtype):
    """msda_packed_attention_bwd gives the bits of the torch functions, which call the entry with a buffer, and leaves the
    statistics' first two entries, so that a second call behind it gives them again."""
    import ctypes

    from rfdetr_jax_amd import _native

    off = _int([0, 70, 200])
    q, k, v, g = _normal(35, dtype, (200, 4, 64), (200, 2, 64), (200, 2, 64), (200, 4, 64))
    out, (stats, rest) = packed_attention_forward(q, k, v, off)
    want = packed_attention_backward(q, k, v, out, (stats, rest), g, off)
    lib, code, dims = _native.lib(), _native.DTYPE_BF16 if dtype == torch.bfloat16 else _native.DTYPE_F32, (2, 200, 200, 4, 2, 64)
    nbytes = lib.msda_packed_attention_bwd_workspace_size(code, *dims)
    ws = _native.workspace(nbytes, q.device)
    ptr = [ctypes.c_void_p(None if x is None else x.data_ptr()) for x in (q, k, v, out, rest, stats, g, off, ws)]
    for _ in range(2):
        grads = [torch.full_like(x, float("nan")) for x in (q, k, v)]
        strides = (ctypes.c_int64 * 16)(*(s for x in (q, k, v, out, g, *grads) for s in x.stride()[:2]))
        rc = lib.msda_packed_attention_bwd(*ptr[:7], code, *(ctypes.c_void_p(x.data_ptr()) for x in grads), ptr[7], ptr[7], None, *dims, strides, 1,
                                           64 ** -0.5, ptr[8], nbytes, ctypes.c_void_p(torch.cuda.current_stream().cuda_stream))
        _native.check(rc)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(grads, want))
