"""Packed attention with shaped scores (cap, slopes, window, prefix) on an MI355X, against the float64 oracle.

Tolerances are the oracle's ``bounds``: element by element, from half a step of the type for each weight, its gradient
and result, 2^-24 for each term of an f32 sum, and the error of the tanh.
"""

from __future__ import annotations

import sys

import numpy as np
import pytest
import torch

from oracle import packed_attention_ref as PA
from oracle import shaped_attention_ref as SA
from rfdetr_jax_amd import packed_attention, packed_attention_backward, packed_attention_forward, rotary_embed

pytestmark = pytest.mark.gpu
HALF_STEP = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}
TYPES = pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])


def _dev():
    assert torch.cuda.is_available(), "GPU tests need a visible MI355X"
    return torch.device("cuda:0")


def _int(x):
    return None if x is None else torch.tensor([int(i) for i in x], dtype=torch.int32, device=_dev())


def _np(t):
    return t.detach().double().cpu().numpy()


def _normal(seed, dtype, *shapes):
    g = torch.Generator().manual_seed(seed)
    return [torch.randn(s, generator=g).to(dtype).to(_dev()) for s in shapes]


def _options(causal=True, cap=None, slopes=None, window=None, prefixes=None):
    kw = dict(cap=cap, window=window, prefix_lengths=_int(prefixes))
    kw["slopes"] = None if slopes is None else torch.tensor(slopes, dtype=torch.float32, device=_dev())
    if slopes is not None:
        slopes = _np(kw["slopes"])
    return kw, SA.Shape(causal, None, cap, slopes, window, prefixes)


def _within(got, want, bound, what):
    got = _np(got)
    assert got.shape == want.shape, what
    assert np.isfinite(got).all(), f"{what}: not finite"
    over = np.abs(got - want) - bound
    at = np.unravel_index(np.argmax(over), over.shape)
    assert over[at] <= 0, f"{what}: off by {abs(got[at] - want[at]):.3e} at {at}, {bound[at]:.3e} allowed"


def _compare(q, k, v, g, got, seqs, shape):
    arrays = [_np(x) for x in (q, k, v, g)]
    want = [SA.attention(*arrays[:3], seqs, shape), *SA.attention_vjp(*arrays, seqs, shape)]
    bound = SA.bounds(*arrays, seqs, HALF_STEP[q.dtype], shape)
    for name, x, w, b in zip(("out", "grad_q", "grad_k", "grad_v"), got, want, bound):
        if x is not None:
            _within(x, w, b, name)


def _run(q, k, v, g, offsets, key_offsets=None, key_lengths=None, causal=True, **kw):
    leaves = [x.detach().requires_grad_(True) for x in (q, k, v)]
    out = packed_attention(*leaves, offsets, key_offsets, key_lengths, causal, **kw)
    assert out.shape == q.shape and out.dtype == q.dtype
    return (out, *torch.autograd.grad(out, leaves, g))


#      lengths, keys, heads, key heads, head dim
SHAPES = {
    "one_token": ([1], [1], 1, 1, 32),
    "ragged": ([5, 64, 1, 130, 33, 0, 63], None, 4, 2, 64),
    "odd_group": ([43, 7, 190], None, 6, 2, 128),
    "one_key_head": ([200, 29], None, 8, 1, 64),
    "dim8": ([170, 3], None, 2, 2, 8),
    "dim40": ([65, 131], None, 3, 1, 40),
    "dim96": ([229, 40], None, 2, 1, 96),
    "more_keys": ([3, 70, 0, 20], [200, 170, 5, 65], 4, 2, 64),
    "fewer_keys": ([40, 9, 230], [10, 0, 127], 4, 2, 32),  # rows before the first key
}


def _slopes(h):
    return [0.5 ** (i % 5) * (-0.25 if i == 3 else 1.0) for i in range(h)]


def _prefixes(keys):
    return [m * (i + 1) % (m + 3) if i % 3 else m // 2 for i, m in enumerate(keys)]


KINDS = {
    "cap": lambda h, keys: dict(cap=30.0),                   # near its line
    "low_cap": lambda h, keys: dict(cap=0.75),               # far beyond it
    "slopes": lambda h, keys: dict(slopes=_slopes(h)),
    "window1": lambda h, keys: dict(window=1),
    "window70": lambda h, keys: dict(window=70),
    "far_window": lambda h, keys: dict(window=2 ** 31 - 1),  # no bound
    "prefix": lambda h, keys: dict(prefixes=_prefixes(keys)),
    "all": lambda h, keys: dict(cap=2.0, slopes=_slopes(h), window=40, prefixes=_prefixes(keys)),
    "open": lambda h, keys: dict(causal=False, cap=5.0, window=33, slopes=_slopes(h)),
}


@TYPES
@pytest.mark.parametrize("kind", sorted(KINDS))
@pytest.mark.parametrize("name", sorted(SHAPES))
def test_against_oracle(name, kind, dtype):
    lengths, keys, h, hk, d = SHAPES[name]
    keys = lengths if keys is None else keys
    sys.stderr.write(f"[gpu] shaped attention {name} {kind} {dtype}\n")
    off, koff = np.cumsum([0, *lengths]), np.cumsum([0, *keys])
    q, k, v, g = _normal(5, dtype, (off[-1], h, d), (koff[-1], hk, d), (koff[-1], hk, d), (off[-1], h, d))
    kw, shape = _options(**KINDS[kind](h, keys))
    got = _run(q, k, v, g, _int(off), _int(koff), causal=shape.causal, **kw)
    _compare(q, k, v, g, got, PA.sequences(off, koff), shape)


@TYPES
@pytest.mark.parametrize("heads", [(8, 1), (4, 4), (16, 2)], ids=["8to1", "4to4", "16to2"])
@pytest.mark.parametrize("new", [1, 7], ids=["one_token", "chunk"])
def test_tokens_over_a_cache(new, heads, dtype):
    """New tokens over caches of different fill, whose keys are split over workgroups, with and without a window;
    unfilled rows, and in the windowed call those before the window, hold NaN."""
    h, hk = heads
    room, fill, d, window = 2500, [2500, 1, 63, 0, 1999, 64], 128, 700
    lengths = [min(new, max(m, 1)) for m in fill]
    lengths[4] = 0
    off, koff = np.cumsum([0, *lengths]), np.arange(len(fill) + 1) * room
    q, k, v, g = _normal(10, dtype, (off[-1], h, d), (koff[-1], hk, d), (koff[-1], hk, d), (off[-1], h, d))
    seqs = PA.sequences(off, koff, fill)
    for options in (dict(cap=4.0), dict(cap=20.0, slopes=_slopes(h), window=window)):
        kw, shape = _options(**options)
        for i, m in enumerate(fill):
            k[koff[i] + m:koff[i + 1]] = v[koff[i] + m:koff[i + 1]] = float("nan")
            if shape.window:
                n = lengths[i]
                gone = max(m - max(n, 1) - window + 1, 0)
                k[koff[i]:koff[i] + gone] = v[koff[i]:koff[i] + gone] = float("nan")
        clean = [torch.nan_to_num(x) for x in (k, v)]
        out, saved = packed_attention_forward(q, k, v, _int(off), _int(koff), _int(fill), **kw)
        assert torch.equal(out, packed_attention(q, k, v, _int(off), _int(koff), _int(fill), **kw))
        grads = packed_attention_backward(q, k, v, out, saved, g, _int(off), _int(koff), _int(fill), **kw)
        _compare(q, *clean, g, (out, *grads), seqs, shape)


@TYPES
def test_long_rows_with_a_window(dtype):
    """A window of many tiles over a longer sequence: tiles are skipped on both sides, and the key side's rows are shared."""
    q, k, v, g = _normal(21, dtype, (1500, 2, 64), (1500, 1, 64), (1500, 1, 64), (1500, 2, 64))
    for options in (dict(window=300), dict(window=129, cap=8.0, causal=False), dict(window=1000, prefixes=[900])):
        kw, shape = _options(**options)
        got = _run(q, k, v, g, _int([0, 1500]), causal=shape.causal, **kw)
        _compare(q, k, v, g, got, PA.sequences([0, 1500]), shape)


@TYPES
def test_infinities_and_nan_of_unseen_pairs(dtype):
    """Rows that hold no finite number beyond a window, behind a prefix and above the diagonal change nothing for the
    queries that do not see them; those that see a value get it."""
    off = [0, 260]
    q, k, v, g = _normal(22, dtype, (260, 2, 64), (260, 1, 64), (260, 1, 64), (260, 2, 64))
    for options in (dict(window=50), dict(prefixes=[70], cap=3.0), dict(window=20, causal=False, slopes=[1.0, 0.1])):
        kw, shape = _options(**options)
        want = packed_attention(q, k, v, _int(off), causal=shape.causal, **kw)
        arrays = [_np(x) for x in (q, k)]
        seen = shape.scores(arrays[0][:, 0], arrays[1][:, 0], 0, 0)[4][:, 150]
        seen = torch.tensor(seen, device=_dev())
        for value in (float("nan"), float("inf"), -float("inf")):
            vv = v.clone()
            vv[150] = value
            got = packed_attention(q, k, vv, _int(off), causal=shape.causal, **kw)
            assert torch.equal(got[~seen], want[~seen])
            assert torch.isnan(got[seen]).all() if value != value else (got[seen] == value).all()
            kk = k.clone()
            kk[150] = value
            got = _run(q, kk, v, g, _int(off), causal=shape.causal, **kw)
            assert torch.equal(got[0][~seen], want[~seen])
            assert torch.isfinite(got[1][~seen]).all() and torch.isnan(got[1][seen]).all()
            assert torch.isfinite(got[3][:100]).all() if shape.causal and shape.window else True
            # a query that is not finite: keys that it does not see keep their gradients
            qq = q.clone()
            qq[150] = value
            got = _run(qq, k, v, g, _int(off), causal=shape.causal, **kw)
            mine = torch.tensor(shape.scores(arrays[0][:, 0], arrays[1][:, 0], 0, 0)[4][150], device=_dev())
            assert torch.isfinite(got[2][~mine]).all() and torch.isfinite(got[3][~mine]).all() and torch.isnan(got[2][mine]).all()


@TYPES
def test_without_options_it_is_the_plain_call(dtype):
    """Options that change nothing give the plain call's results within the roundings of both."""
    off = [0, 100, 333]
    q, k, v, g = _normal(23, dtype, (333, 4, 64), (333, 2, 64), (333, 2, 64), (333, 4, 64))
    plain = _run(q, k, v, g, _int(off))
    kw, shape = _options(window=333)
    got = _run(q, k, v, g, _int(off), **kw)
    _compare(q, k, v, g, got, PA.sequences(off), shape)
    again = _run(q, k, v, g, _int(off), cap=None, slopes=None, window=None, prefix_lengths=None)
    assert all(torch.equal(a, b) for a, b in zip(plain, again))
    kw, shape = _options(prefixes=[0, -5])
    _compare(q, k, v, g, _run(q, k, v, g, _int(off), **kw), PA.sequences(off), SA.Shape())


def test_gradients_against_differences():
    """f32, directional, along the oracle's own central differences: scores on both sides of the cap."""
    off, h = [0, 90], 2
    q, k, v, g = _normal(24, torch.float32, (90, h, 32), (90, 1, 32), (90, 1, 32), (90, h, 32))
    kw, shape = _options(cap=1.0, slopes=[0.1, 0.0], window=60)
    got = _run(q, k, v, g, _int(off), **kw)
    arrays, seqs = [_np(x) for x in (q, k, v, g)], PA.sequences(off)
    r = np.random.default_rng(0)
    for i in range(3):
        way = r.standard_normal(arrays[i].shape)
        ends = []
        for sign in (1, -1):
            moved = list(arrays)
            moved[i] = moved[i] + sign * 1e-5 * way
            ends.append((SA.attention(*moved[:3], seqs, shape) * arrays[3]).sum())
        bound = SA.bounds(*arrays, seqs, 2.0 ** -24, shape)[i + 1]
        # the differences' own error: their third-order term, below 1e-10 of sums of this size, and 2^-52 of the sums / 1e-5
        assert abs((ends[0] - ends[1]) / 2e-5 - (_np(got[i + 1]) * way).sum()) <= (bound * np.abs(way)).sum() + 1e-6


@TYPES
def test_the_python_path_gives_the_same(dtype, monkeypatch):
    """The C++ autograd function and the Python one, and the functions without autograd, give the same bits."""
    from rfdetr_jax_amd import _native

    off = [0, 60, 190]
    q, k, v, g = _normal(25, dtype, (190, 4, 64), (190, 2, 64), (190, 2, 64), (190, 4, 64))
    kw, _ = _options(cap=5.0, slopes=_slopes(4), window=64, prefixes=[30, 50])
    want = _run(q, k, v, g, _int(off), **kw)
    out, saved = packed_attention_forward(q, k, v, _int(off), **kw)
    got = (out, *packed_attention_backward(q, k, v, out, saved, g, _int(off), **kw))
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    monkeypatch.setattr(_native, "binding", lambda: _native._NoBinding)
    got = _run(q, k, v, g, _int(off), **kw)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    kw["prefix_lengths"] = kw["prefix_lengths"].long()  # and what only the Python path takes
    kw["slopes"] = torch.stack([kw["slopes"]] * 2, 1)[:, 0]
    got = _run(q, k, v, g, _int(off), **kw)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@TYPES
def test_in_a_graph_with_other_lengths(dtype):
    """One captured forward and backward, replayed with other lengths, prefixes and slopes and other eager work between."""
    q, k, v, g = _normal(16, dtype, (300, 4, 64), (300, 2, 64), (300, 2, 64), (300, 4, 64))
    off, prefixes = _int([0, 100, 300]), _int([40, 60])
    slopes = torch.tensor(_slopes(4), device=_dev())
    cq, ck, cv = _normal(17, dtype, (2, 4, 64), (4000, 2, 64), (4000, 2, 64))
    coff, ckoff, fill = _int([0, 1, 2]), _int([0, 2000, 4000]), _int([2000, 5])

    def work():
        kw = dict(cap=6.0, slopes=slopes, window=90, prefix_lengths=prefixes)
        out, stats = packed_attention_forward(q, k, v, off, **kw)
        return (out, *packed_attention_backward(q, k, v, out, stats, g, off, **kw), packed_attention(cq, ck, cv, coff, ckoff, fill, cap=6.0, window=1500))

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
        prefixes.add_(11)
        slopes.mul_(0.5)
        q.mul_(-0.5)
        eager = work()
        torch.cuda.synchronize()
        for x in outs:
            x.fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, eager)), (lengths, filled)


def test_offsets_that_do_not_rise_stay_in_bounds():
    q, k, v, g = _normal(13, torch.float32, (150, 4, 32), (300, 2, 32), (300, 2, 32), (150, 4, 32))
    for off, koff, lengths, prefixes in (([0, 150, 20, 150], [0, 300, 10, 300], None, [2 ** 31 - 1, -2 ** 31, 5]),
                                         ([-5, 40, 1000, 2000], [-9, 100, 400, 9000], [900, -3, 50], [1, 2, 3]),
                                         ([150, 0, 0, 0], [300, 0, 0, 0], [3, 3, 3], [2 ** 31 - 1] * 3)):
        for window in (None, 30, 2 ** 31 - 1):
            kw, _ = _options(cap=2.0, slopes=_slopes(4), window=window, prefixes=prefixes)
            got = _run(q, k, v, g, _int(off), _int(koff), _int(lengths), **kw)
            assert [x.shape for x in got] == [q.shape, q.shape, k.shape, v.shape]
    off, koff = [0, 100, 150], [0, 200, 300]
    kw, shape = _options(cap=2.0, window=30)
    _compare(q, k, v, g, _run(q, k, v, g, _int(off), _int(koff), **kw), PA.sequences(off, koff), shape)


@TYPES
def test_image_and_text_with_rotary_positions(dtype):
    """As they are used together: an image whose patches see each other and a text behind it, positions on two axes, then
    the text's last token again over a cache."""
    h, hk, d, image, text = 4, 2, 64, 49, 30
    n = image + text
    (qkv,) = _normal(18, dtype, (n, h + 2 * hk, d))
    grid = torch.cartesian_prod(torch.arange(7), torch.arange(7))
    pos = torch.cat([grid, torch.arange(7, 7 + text)[:, None].expand(text, 2)]).to(torch.int32).to(_dev())
    q, k = rotary_embed(qkv[:, :h], qkv[:, h:h + hk], pos, (16, 16))
    v = qkv[:, h + hk:]
    kw, shape = _options(cap=8.0, prefixes=[image])
    out = packed_attention(q, k, v, _int([0, n]), **kw)
    arrays, seqs = [_np(x) for x in (q, k, v)], PA.sequences([0, n])
    bound = SA.bounds(*arrays, np.zeros(arrays[0].shape), seqs, HALF_STEP[dtype], shape)
    want = SA.attention(*arrays, seqs, shape)
    _within(out, want, bound[0], "prompt")
    cache = [torch.cat([x, torch.full_like(x, float("nan"))]) for x in (k, v)]
    last = packed_attention(q[-1:], *cache, _int([0, 1]), _int([0, 2 * n]), _int([n]), **kw)
    _within(last, want[-1:], bound[0][-1:], "token")


#      lengths, keys, heads, key heads, head dim
WIDE = {
    "thousands": ([int(i * 7919 % 4) for i in range(3000)], None, 2, 1, 8),  # searched, not counted
    "sixty_four_to_a_head": ([40, 3], [150, 3], 64, 1, 64),
    "thirty_three_to_a_head": ([30, 66], None, 66, 2, 32),
    "one_token_in_many": ([0] * 100 + [1] + [0] * 100, [0] * 100 + [333] + [0] * 100, 64, 2, 128),
    "long_keys": ([130, 2], [4000, 3000], 2, 1, 128),
    "long_rows": ([3100, 2], None, 2, 1, 32),
}


@TYPES
@pytest.mark.parametrize("name", sorted(WIDE))
def test_many_sequences_wide_groups_and_long_keys(name, dtype):
    lengths, keys, h, hk, d = WIDE[name]
    keys = lengths if keys is None else keys
    sys.stderr.write(f"[gpu] shaped attention {name} {dtype}\n")
    off, koff = np.cumsum([0, *lengths]), np.cumsum([0, *keys])
    q, k, v, g = _normal(26, dtype, (off[-1], h, d), (koff[-1], hk, d), (koff[-1], hk, d), (off[-1], h, d))
    for options in (dict(cap=3.0, slopes=_slopes(h), prefixes=_prefixes(keys)), dict(window=100, slopes=_slopes(h))):
        kw, shape = _options(**options)
        got = _run(q, k, v, g, _int(off), _int(koff), **kw)
        _compare(q, k, v, g, got, PA.sequences(off, koff), shape)


@TYPES
def test_caps_of_every_size(dtype):
    """From one that flattens everything to one that changes nothing, beside scales of other sizes: far, near and both in
    a block."""
    off = [0, 100, 171]
    q, k, v, g = _normal(27, dtype, (171, 2, 64), (171, 1, 64), (171, 1, 64), (171, 2, 64))
    for cap, scale in ((2.0 ** -32, None), (0.01, None), (1.0, 3.0), (4.0, 1.0), (1000.0, 2.0), (2.0 ** 20, None), (2.0 ** 32, 0.5), (30.0, 2.0 ** -40)):
        kw, shape = _options(cap=cap)
        shape.scale = scale
        got = _run(q, k, v, g, _int(off), scale=scale, **kw)
        _compare(q, k, v, g, got, PA.sequences(off), shape)


@TYPES
def test_layouts_and_one_gradient_at_a_time(dtype):
    """Slices of a projection, head-major tensors, a cotangent by stride 0; gradients wanted one by one: the same bits."""
    off, h, hk, d = [0, 50, 131], 4, 2, 64
    (qkv,) = _normal(28, dtype, (131, h + 2 * hk, d))
    parts = [qkv[:, :h], qkv[:, h:h + hk], qkv[:, h + hk:]]
    (g,) = _normal(29, dtype, (131, h, d))
    kw, shape = _options(cap=2.0, slopes=_slopes(h), window=60, prefixes=[20, 131])
    want = _run(*(x.contiguous() for x in parts), g, _int(off), **kw)
    _compare(*parts, g, want, PA.sequences(off), shape)
    for other in (parts, [x.transpose(0, 1).contiguous().transpose(0, 1) for x in parts], [x.transpose(1, 2).contiguous().transpose(1, 2) for x in parts]):
        assert all(torch.equal(a, b) for a, b in zip(_run(*other, g, _int(off), **kw), want))
    out, saved = packed_attention_forward(*parts, _int(off), **kw)
    for i in range(3):
        needs = [j == i for j in range(3)]
        got = packed_attention_backward(*parts, out, saved, g, _int(off), needs=needs, **kw)
        assert [x is not None for x in got] == needs and torch.equal(got[i], want[i + 1])
    ones = torch.ones((), dtype=dtype, device=_dev()).expand(131, h, d)
    _compare(*parts, ones, _run(*parts, ones, _int(off), **kw), PA.sequences(off), shape)


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("dim", [8, 16, 32, 40, 64, 80])
def test_gradients_of_few_channels(dim, causal):
    """bf16, scores of four standard deviations: the keys that a row weighs most lie along its query, and what they share
    cancels in the sum of ds k. One rounding of each ds would not cancel: it alone is the result's own rounding again (their
    sum the square root of two of it), times the root of (a^2 + D) / D, a the shared part in standard deviations. So grad_q
    has to be nearer than the square root of two: its own rounding, and delta's error, smaller than that."""
    n, h, hk = 900, 4, 2
    q, k, v, g = _normal(31 + dim, torch.float32, (n, h, dim), (n, hk, dim), (n, hk, dim), (n, h, dim))
    q, k, v, g = (x.bfloat16() for x in (4.0 * q, k, v, g))
    kw, shape = _options(causal=causal, cap=50.0)
    off = np.array([0, n])
    got = _run(q, k, v, g, _int(off), causal=causal, **kw)
    arrays = [_np(x) for x in (q, k, v, g)]
    want = SA.attention_vjp(*arrays, PA.sequences(off, off, None), shape)[0]
    rounded = np.linalg.norm(_np(torch.from_numpy(want).bfloat16()) - want)
    assert np.linalg.norm(_np(got[1]) - want) < 2 ** 0.5 * rounded


@TYPES
@pytest.mark.parametrize("kind", ["all", "cap", "open", "prefix"])
def test_tiles_that_workgroups_share(kind, dtype):
    """Few tiles of queries over many keys, rows in front of the first sequence and behind the last, a sequence without keys
    and one that sees its first keys alone; twice, with the same bits."""
    lengths, keys, h, hk, d = [300, 0, 45, 131], [1900, 7, 0, 1400], 4, 2, 64
    off, koff = np.cumsum([0, *lengths]) + 3, np.cumsum([0, *keys]) + 2
    q, k, v, g = _normal(41, dtype, (off[-1] + 5, h, d), (koff[-1] + 4, hk, d), (koff[-1] + 4, hk, d), (off[-1] + 5, h, d))
    for x, ends in ((q, off), (g, off), (k, koff), (v, koff)):
        x[:ends[0]] = x[ends[-1]:] = float("nan")
    kw, shape = _options(**KINDS[kind](h, keys))
    causal = kind != "open"
    got = _run(q, k, v, g, _int(off), _int(koff), causal=causal, **kw)
    for x, ends in zip(got, (off, off, koff, koff)):
        assert not x[:ends[0]].any() and not x[ends[-1]:].any()
    for a, b in zip(got, _run(q, k, v, g, _int(off), _int(koff), causal=causal, **kw)):
        assert torch.equal(a, b)
    inner, outer = slice(off[0], off[-1]), slice(koff[0], koff[-1])
    _compare(q[inner], k[outer], v[outer], g[inner], [x[s] for x, s in zip(got, (inner, inner, outer, outer))], PA.sequences(off - 3, koff - 2), shape)
