"""The cache in 4 bits (rfdetr_jax_amd.cache4_write, cache4_read, cache4_attention) on an MI355X, against the oracles:
codes and values to the bit, attention within the bounds of shaped_attention_ref for the values that the cache holds."""

from __future__ import annotations

import sys

import numpy as np
import pytest
import torch

from oracle import cache4_ref as C4
from oracle import packed_attention_ref as PA
from oracle import shaped_attention_ref as SA
from rfdetr_jax_amd import (
    Cache4, _native, cache4_attention, cache4_read, cache4_write, new_cache4, norm_rotary_embed, packed_attention,
)

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


def _bytes(cache):
    return [t.cpu().numpy() for t in cache[:4]]


def _random_cache(seed, rows, hk, d):
    """A cache of normal numbers, codes and scales as random as these make them (built here, not by the kernel)."""
    r = np.random.default_rng(seed)
    blocks = (d + 31) // 32
    out = []
    for _ in range(2):
        codes = r.integers(0, 16, (hk, rows, 32 * blocks)).astype(np.uint8)
        codes[..., d:] = 0
        out += [codes[..., 0::2] | codes[..., 1::2] << 4, (126 + r.integers(-2, 2, (hk, rows, blocks))).astype(np.uint8)]
    return Cache4(*(torch.from_numpy(x).to(_dev()) for x in out), d)


def _held(cache):
    """The cache's values, [rows, Hk, D] in float64."""
    b = _bytes(cache)
    return [C4.decode(b[i], b[i + 1], cache.head_dim).transpose(1, 0, 2) for i in (0, 2)]


def _within(got, want, bound, what):
    got = _np(got)
    assert got.shape == want.shape and np.isfinite(got).all(), f"{what}: not finite"
    over = np.abs(got - want) - bound
    at = np.unravel_index(np.argmax(over), over.shape)
    assert over[at] <= 0, f"{what}: off by {abs(got[at] - want[at]):.3e} at {at}, {bound[at]:.3e} allowed"


def _options(causal=True, cap=None, slopes=None, window=None, prefixes=None):
    kw = dict(cap=cap, window=window, prefix_lengths=_int(prefixes), causal=causal)
    kw["slopes"] = None if slopes is None else torch.tensor(slopes, dtype=torch.float32, device=_dev())
    return kw, SA.Shape(causal, None, cap, None if slopes is None else _np(kw["slopes"]), window, prefixes)


def _check(out, q, cache, seqs, shape, few):
    """few: no sequence has more than 16 rows to a key head, whose weights are two bf16 numbers."""
    k, v = (np.nan_to_num(x) for x in _held(cache))
    arrays, u = [_np(q), k, v], HALF_STEP[q.dtype]
    want = SA.attention(*arrays, seqs, shape)
    weights = 2.0 ** -16 if few and u == 2.0 ** -8 else u
    bound = SA.bounds(*arrays, np.zeros(arrays[0].shape), seqs, weights, shape)[0] + u * np.abs(want) * (1 + u)
    _within(out, want, bound, "out")


# ---- writing and reading ----------------------------------------------------------------------


@TYPES
@pytest.mark.parametrize("d", [8, 32, 40, 64, 72, 96, 120, 128])
def test_rows_written_and_read(d, dtype):
    """Packed new tokens at the ends of their sequences' keys: the oracle's bytes there, and the others as they were; read
    back, in both types, the values that the bytes stand for."""
    hk, off, koff, lengths = 3, [2, 7, 7, 20, 26], [5, 20, 30, 60, 64], [9, 4, 25, 4]
    tokens, rows = 29, 70
    k, v = _normal(1, dtype, (tokens, hk, d), (tokens, hk, d))
    k = k * torch.exp(3 * _normal(2, torch.float32, (tokens, hk, 1))[0]).to(dtype)
    k[3, 0, :8] = torch.tensor([6, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0], dtype=dtype)  # ties
    k[3, 0, 8:] = 0
    k[4, 1], v[5, 2] = 0, 1e-38
    v[6, 0] = 3e38
    cache = _random_cache(3, rows, hk, d)
    before = _bytes(cache)
    cache4_write(cache, k, v, _int(off), _int(koff), _int(lengths))
    want, read = [x.copy() for x in before], [np.zeros((tokens, hk, d)) for _ in range(2)]
    for i, (q0, n, k0, m) in enumerate(PA.sequences(off, koff, lengths)):
        for t in range(n):
            place = m - n + t
            if place < 0:
                continue
            for j, x in enumerate((k, v)):
                codes, scales = C4.encode(_np(x[q0 + t]))
                want[2 * j][:, k0 + place], want[2 * j + 1][:, k0 + place] = codes, scales
                read[j][q0 + t] = C4.decode(codes, scales, d)
    for a, b in zip(_bytes(cache), want):
        np.testing.assert_array_equal(a, b)
    for kind in (torch.float32, torch.bfloat16):
        got = cache4_read(cache, tokens, _int(off), _int(koff), _int(lengths), dtype=kind)
        for a, b in zip(got, read):
            assert a.dtype == kind
            np.testing.assert_array_equal(_np(a), b)


@TYPES
def test_every_value_of_a_type_is_rounded_right(dtype):
    """A sweep over mantissas and exponents, ties and their neighbours, against the oracle's bytes."""
    if dtype == torch.bfloat16:
        bits = torch.arange(0, 1 << 16, 3, dtype=torch.int32) << 16
    else:
        r = np.random.default_rng(5)
        ties = np.array([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 7.0], np.float32).view(np.int32)
        near = (ties[None, :] + np.arange(-3, 4)[:, None]).reshape(-1)
        bits = torch.from_numpy(np.concatenate([near, r.integers(0, 1 << 31, 8000)]).astype(np.int32))
    x = bits.view(torch.float32)
    x = x[torch.isfinite(x)]
    rows = x.numel() // 64
    # a row of 64 has two blocks: one with the number beside a 6 and zeros, one as it comes
    x = x[:rows * 64].view(rows, 1, 64)
    beside = torch.zeros(rows, 1, 64)
    beside[..., :31], beside[..., 31] = x[..., :31].clamp(-7, 7), 6.0
    x = torch.cat([beside[..., :32], x[..., 32:]], -1).to(dtype).to(_dev())
    cache = new_cache4(rows, 1, 64, _dev())
    cache4_write(cache, x, x.flip(-1), _int([0, rows]))
    for i, y in ((0, x), (2, x.flip(-1))):
        codes, scales = C4.encode(_np(y).transpose(1, 0, 2))
        np.testing.assert_array_equal(cache[i].cpu().numpy(), codes)
        np.testing.assert_array_equal(cache[i + 1].cpu().numpy(), scales)


@TYPES
def test_infinities_and_nan_are_their_block(dtype):
    d, off = 96, [0, 4]
    k, v = _normal(6, dtype, (4, 2, d), (4, 2, d))
    k[1, 0, 40], v[2, 1, 95], v[2, 1, 3], k[3, 1, 0] = float("nan"), float("inf"), -float("inf"), float("nan")
    cache = new_cache4(4, 2, d, _dev())
    cache4_write(cache, k, v, _int(off))
    for x, got, i in zip((k, v), cache4_read(cache, 4, _int(off), dtype=torch.float32), (0, 2)):
        codes, scales = C4.encode(_np(x).transpose(1, 0, 2))
        np.testing.assert_array_equal(cache[i].cpu().numpy(), codes)
        np.testing.assert_array_equal(cache[i + 1].cpu().numpy(), scales)
        np.testing.assert_array_equal(_np(got), C4.decode(codes, scales, d).transpose(1, 0, 2))
        bad = ~torch.isfinite(x.float()).view(4, 2, 3, 32).all(-1)
        assert torch.equal(torch.isnan(got).view(4, 2, 3, 32).all(-1), bad) and torch.equal(torch.isnan(got).view(4, 2, 3, 32).any(-1), bad)


@TYPES
def test_layouts_and_many_sequences(dtype):
    """Slices of a projection, head-major tensors, rows off their boundaries; 300 sequences of 0 to 3 tokens; no tokens."""
    hk, d = 2, 64
    counts = [i * 7919 % 4 for i in range(300)]
    off = np.cumsum([0, *counts])
    (qkv,) = _normal(7, dtype, (off[-1], 3 * hk, d))
    parts = [qkv[:, hk:2 * hk], qkv[:, 2 * hk:]]
    koff, fill = np.arange(301) * 5, [c + i % 2 for i, c in enumerate(counts)]
    caches = []
    shifted = [torch.empty(x.numel() + 1, dtype=dtype, device=_dev())[1:].view(x.shape).copy_(x) for x in parts]
    for k, v in (parts, [x.transpose(0, 1).contiguous().transpose(0, 1) for x in parts], shifted, [x.transpose(1, 2).contiguous().transpose(1, 2) for x in parts]):
        cache = new_cache4(1500, hk, d, _dev())
        cache4_write(cache, k, v, _int(off), _int(koff), _int(fill))
        caches.append(_bytes(cache))
        got = cache4_read(cache, off[-1], _int(off).long(), _int(koff), _int(fill))
        for a, x in zip(got, parts):
            np.testing.assert_array_equal(_np(a), C4.decode(*C4.encode(_np(x)), d))
    for other in caches[1:]:
        assert all((a == b).all() for a, b in zip(caches[0], other))
    cache4_write(cache, parts[0][:0], parts[1][:0], _int([0]), _int([0]))
    assert [x.shape[0] for x in cache4_read(cache, 0, _int([0, 0]), _int([0, 4]))] == [0, 0]
    assert not any(x.any() for x in cache4_read(cache, 5, _int([0]), _int([0])))


def test_wrong_places_stay_in_bounds():
    """Offsets that fall, are negative or too large, lengths past the room: the calls end, and a right one is right."""
    k, v, q = _normal(8, torch.float32, (50, 2, 32), (50, 2, 32), (50, 4, 32))
    cache = _random_cache(9, 60, 2, 32)
    for off, koff, lengths in (([0, 50, 20, 50], [0, 60, 10, 60], None), ([-5, 20, 1000, 2000], [-9, 30, 400, 9000], [900, -3, 50]),
                               ([50, 0, 0, 0], [60, 0, 0, 0], [3, 3, 3]), ([0, 2 ** 31 - 1, -2 ** 31, 7], [2 ** 31 - 1, 0, 0, 5], [2 ** 31 - 1] * 3)):
        cache4_write(cache, k, v, _int(off), _int(koff), _int(lengths))
        assert cache4_read(cache, 50, _int(off), _int(koff), _int(lengths))[0].shape == (50, 2, 32)
        for many in (1, 100):  # both kernels
            o, ko = _int([*off, *([off[-1]] * many)]), _int([*koff, *([koff[-1]] * many)])
            ln = None if lengths is None else _int([*lengths, *([0] * many)])
            for kw in ({}, dict(window=9, cap=2.0, prefix_lengths=_int([2 ** 31 - 1] * (3 + many)))):
                assert cache4_attention(q, cache, o, ko, ln, **kw).shape == q.shape
    cache4_write(cache, k, v, _int([0, 50]), _int([10, 60]))
    codes, scales = C4.encode(_np(k).transpose(1, 0, 2))
    np.testing.assert_array_equal(cache.keys[:, 10:].cpu().numpy(), codes)
    np.testing.assert_array_equal(cache.key_scales[:, 10:].cpu().numpy(), scales)


# ---- attention --------------------------------------------------------------------------------


#      new tokens, keys, room, heads, key heads, head dim
SHAPES = {
    "one_key": ([1], [1], 4, 1, 1, 32),
    "one_token": ([1], [700], 1024, 8, 2, 64),
    "tokens": ([1] * 9, [2500, 1, 63, 0, 1999, 64, 65, 128, 1025], 2500, 8, 2, 128),
    "all_heads": ([1, 1], [300, 77], 300, 4, 4, 128),
    "one_key_head": ([1, 2], [300, 1500], 1500, 8, 1, 96),
    "sixty_four_to_a_head": ([1, 0, 1], [130, 50, 700], 700, 64, 1, 64),
    "dim40": ([2, 1], [90, 130], 200, 3, 1, 40),
    "dim8": ([1, 1], [70, 3], 80, 2, 2, 8),
    "dim72": ([3, 1], [70, 200], 200, 2, 2, 72),
    "chunks": ([200, 33, 1], [1500, 33, 999], 1600, 4, 2, 128),   # rows in tiles
    "chunks96": ([150, 7], [300, 500], 500, 6, 2, 96),
    "chunks40": ([40, 130], [400, 130], 400, 3, 1, 40),
    "chunks32": ([100], [333], 400, 2, 1, 32),
    "more_tokens_than_keys": ([9, 200], [4, 100], 128, 2, 1, 64),  # rows that see no key
    "mixed": ([30, 1, 1, 1, 1, 1, 1, 1], [2000, 5, 100, 999, 64, 1, 70, 300], 2048, 4, 2, 64),  # few rows on average
}
KINDS = {
    "plain": lambda h, keys: {},
    "open": lambda h, keys: dict(causal=False),
    "cap": lambda h, keys: dict(cap=3.0),
    "slopes_window": lambda h, keys: dict(slopes=[0.5 ** (i % 4) for i in range(h)], window=70),
    "prefix": lambda h, keys: dict(prefixes=[m // 2 for m in keys], cap=20.0),
    "all": lambda h, keys: dict(cap=2.0, slopes=[0.1 * (i % 3) - 0.05 for i in range(h)], window=333, prefixes=[m - i for i, m in enumerate(keys)]),
}


@TYPES
@pytest.mark.parametrize("kind", sorted(KINDS))
@pytest.mark.parametrize("name", sorted(SHAPES))
def test_attention_against_oracle(name, kind, dtype):
    lengths, fill, room, h, hk, d = SHAPES[name]
    sys.stderr.write(f"[gpu] cache in 4 bits {name} {kind} {dtype}\n")
    off, koff = np.cumsum([0, *lengths]), np.arange(len(fill) + 1) * room
    cache = _random_cache(10, koff[-1], hk, d)
    (q,) = _normal(11, dtype, (off[-1] + 3, h, d))  # rows behind the last sequence
    q[off[-1]:] = float("nan")
    kw, shape = _options(**KINDS[kind](h, fill))
    out = cache4_attention(q, cache, _int(off), _int(koff), _int(fill), **kw)
    assert out.dtype == dtype and not out[off[-1]:].any()
    few = max(lengths) * h // hk <= 16
    _check(out[:off[-1]], q[:off[-1]], cache, PA.sequences(off, koff, fill), shape, few)


@TYPES
@pytest.mark.parametrize("name", ["tokens", "chunks", "mixed"])
def test_rows_before_and_behind_and_blocks_that_are_not_finite(name, dtype):
    """Unfilled rows, and ones beyond a window, hold blocks of NaN and change nothing; a bad block of a key that is seen makes
    the row NaN, one of a value its channels."""
    lengths, fill, room, h, hk, d = SHAPES[name]
    off, koff = np.cumsum([0, *lengths]) + 2, np.arange(len(fill) + 1) * room
    cache = _random_cache(12, koff[-1], hk, d)
    (q,) = _normal(13, dtype, (off[-1], h, d))
    for options in ({}, dict(window=100, cap=5.0)):
        kw, shape = _options(**options)
        args = (_int(off), _int(koff), _int(fill))
        want = cache4_attention(q, cache, *args, **kw)
        assert not want[:2].any()
        seqs = PA.sequences(off, koff, fill)
        _check(want, q, cache, seqs, shape, False)
        bad = Cache4(*(t.clone() for t in cache[:4]), d)
        for (q0, n, k0, m) in seqs:
            bad.key_scales[:, k0 + m:k0 + room] = 255
            bad.value_scales[:, k0 + m:k0 + room] = 255
            gone = max(m - max(n, 1) - 99, 0) if options else 0
            bad.key_scales[:, k0:k0 + gone] = 255
            bad.value_scales[:, k0:k0 + gone] = 255
        assert torch.equal(cache4_attention(q, bad, *args, **kw), want)
        at = next(i for i, (q0, n, k0, m) in enumerate(seqs) if n and m > 60)
        q0, n, k0, m = seqs[at]
        key = m - 1 - min(20, m - 1)
        sees = torch.tensor([(key <= t + m - n) and (not options or t + m - n - key < 100) for t in range(n)], device=_dev())
        rows = torch.zeros(off[-1], dtype=torch.bool, device=_dev())
        rows[q0:q0 + n] = sees
        for which in ("value_scales", "key_scales"):
            one = Cache4(*(t.clone() for t in cache[:4]), d)
            getattr(one, which)[hk - 1, k0 + key, 1] = 255
            got = cache4_attention(q, one, *args, **kw)
            heads = slice((hk - 1) * (h // hk), h)
            assert torch.equal(got[~rows], want[~rows]) and torch.equal(got[:, :heads.start], want[:, :heads.start])
            hit = got[rows][:, heads]
            if which == "key_scales":
                assert torch.isnan(hit).all()
            else:
                assert torch.isnan(hit[..., 32:64]).all()
                rest = [c for c in range(d) if not 32 <= c < 64]
                assert torch.equal(hit[..., rest], want[rows][:, heads][..., rest])


@TYPES
@pytest.mark.parametrize("name", ["tokens", "chunks", "chunks96", "mixed"])
def test_memory_that_nothing_wrote(name, dtype):
    """Any bytes where no key is seen, scales of no finite block (253 and more) among them."""
    lengths, fill, room, h, hk, d = SHAPES[name]
    off, koff = np.cumsum([0, *lengths]), np.arange(len(fill) + 1) * room
    cache = _random_cache(22, koff[-1], hk, d)
    (q,) = _normal(23, dtype, (off[-1], h, d))
    g = torch.Generator().manual_seed(24)
    kw, _ = _options(window=100)
    args = (_int(off), _int(koff), _int(fill))
    want = cache4_attention(q, cache, *args, **kw)
    for scale in (0, 253, 254, None):
        other = Cache4(*(t.clone() for t in cache[:4]), d)
        for (q0, n, k0, m) in PA.sequences(off, koff, fill):
            for rows in (slice(k0 + m, k0 + room), slice(k0, k0 + max(m - max(n, 1) - 99, 0))):
                for t in other[:4]:
                    t[:, rows] = torch.randint(0, 256, t[:, rows].shape, generator=g, dtype=torch.uint8).to(_dev())
                if scale is not None:
                    other.key_scales[:, rows] = other.value_scales[:, rows] = scale
        assert torch.equal(cache4_attention(q, other, *args, **kw), want), scale


@TYPES
def test_large_scores(dtype):
    """Scores that rise and fall by hundreds along the keys, in both kernels."""
    d, m = 64, 900
    cache = _random_cache(14, m, 1, d)
    for flip in (False, True):
        ramp = torch.linspace(0, 9, m, device=_dev()).round().to(torch.uint8)
        ramp = ramp.flip(0) if flip else ramp
        steep = Cache4(cache.keys, cache.key_scales - 4 + ramp[None, :, None], cache.values, cache.value_scales, d)
        for n in (2, 40):
            (q,) = _normal(15, dtype, (n, 4, d))
            out = cache4_attention(q, steep, _int([0, n]), _int([0, m]))
            _check(out, q, steep, [(0, n, 0, m)], SA.Shape(), n == 2)


@TYPES
def test_layouts_and_the_python_path(dtype, monkeypatch):
    lengths, fill, room, h, hk, d = SHAPES["tokens"]
    off, koff = np.cumsum([0, *lengths]), np.arange(len(fill) + 1) * room
    cache = _random_cache(16, koff[-1], hk, d)
    (qkv,) = _normal(17, dtype, (off[-1], h + 2, d))
    q = qkv[:, 1:h + 1]
    args = (_int(off), _int(koff), _int(fill))
    kw, _ = _options(cap=4.0, slopes=[0.1] * h, window=900, prefixes=[3] * len(fill))
    want = [cache4_attention(q, cache, *args), cache4_attention(q, cache, *args, **kw)]
    other = torch.empty(q.numel() + 1, dtype=dtype, device=_dev())[1:].view(q.shape).copy_(q)
    for x in (q.contiguous(), q.transpose(0, 1).contiguous().transpose(0, 1), other, q.transpose(1, 2).contiguous().transpose(1, 2)):
        assert torch.equal(cache4_attention(x, cache, *args), want[0])
    assert torch.equal(cache4_attention(q, cache, *args, scale=d ** -0.5), want[0])
    caches = [new_cache4(koff[-1], hk, d, _dev()) for _ in range(2)]
    k, v = _normal(18, dtype, (off[-1], hk, d), (off[-1], hk, d))
    cache4_write(caches[0], k, v, *args)
    reads = cache4_read(caches[0], off[-1], *args)
    monkeypatch.setattr(_native, "binding", lambda: _native._NoBinding)
    assert torch.equal(cache4_attention(q, cache, *args), want[0]) and torch.equal(cache4_attention(q, cache, *args, **kw), want[1])
    cache4_write(caches[1], k, v, *args)
    assert all(torch.equal(a, b) for a, b in zip(caches[0][:4], caches[1][:4]))
    assert all(torch.equal(a, b) for a, b in zip(reads, cache4_read(caches[1], off[-1], *args)))


def test_a_cache_past_32_bits():
    """Codes of a head that begin behind 2^32 bytes."""
    hk, d, rows = 3, 128, (1 << 25) + 640
    cache = Cache4(*(torch.empty((hk, rows, n), dtype=torch.uint8, device=_dev()) for n in (64, 4) * 2), d)
    m, first = 300, rows - 310
    k, v = _normal(19, torch.bfloat16, (m, hk, d), (m, hk, d))
    koff = _int([first, rows])
    cache4_write(cache, k, v, _int([0, m]), koff, _int([m]))
    small = new_cache4(m, hk, d, _dev())
    cache4_write(small, k, v, _int([0, m]))
    assert all(torch.equal(a[:, first:first + m], b) for a, b in zip(cache[:4], small[:4]))
    assert all(torch.equal(a, b) for a, b in zip(cache4_read(cache, m, _int([0, m]), koff, _int([m])), cache4_read(small, m, _int([0, m]))))
    for n in (1, 50):
        (q,) = _normal(20, torch.bfloat16, (n, 2 * hk, d))
        out = cache4_attention(q, cache, _int([0, n]), koff, _int([m]))
        _check(out, q, small, [(0, n, 0, m)], SA.Shape(), n == 1)


def test_refusals_on_a_gpu():
    cache = new_cache4(16, 2, 64, _dev())
    k, q = _normal(21, torch.bfloat16, (4, 2, 64), (4, 4, 64))
    off = _int([0, 4])
    for args, error, text in (((cache, k.half(), k, off), TypeError, "dtype"), ((cache, k, k.float(), off), TypeError, "one type"),
                              ((cache, k[:, :1], k, off), ValueError, "must be"), ((cache, k.cpu(), k, off), ValueError, "cache on"),
                              ((cache, k, k, off.float()), TypeError, "int32"), ((cache, k, k, off, _int([0])), ValueError, "key_offsets"),
                              ((cache, k.detach().requires_grad_(True), k, off), ValueError, "gradient"),
                              ((cache._replace(keys=cache.keys[:, ::2]), k, k, off), ValueError, "contiguous|must be"),
                              ((cache._replace(head_dim=96), k, k, off), ValueError, "must be"),
                              ((cache._replace(values=cache.values.int()), k, k, off), TypeError, "uint8")):
        with pytest.raises(error, match=text):
            cache4_write(*args)
    for args, kw, error, text in (((q.half(), cache, off), {}, TypeError, "dtype"), ((q[:, :3], cache, off), {}, ValueError, "divide"),
                                  ((q[..., :32], cache, off), {}, ValueError, "64"), ((q.cpu(), cache, off), {}, ValueError, "cache on"),
                                  ((q.detach().requires_grad_(True), cache, off), {}, ValueError, "gradient"),
                                  ((q, cache, off), dict(cap=-1.0), ValueError, "cap"), ((q, cache, off), dict(window=0), ValueError, "window"),
                                  ((q, cache, off), dict(scale=0.0), ValueError, "scale"), ((q, cache, off, None, _int([1, 2])), {}, ValueError, "key_lengths")):
        with pytest.raises(error, match=text):
            cache4_attention(*args, **kw)
    with torch.no_grad():
        cache4_write(cache, k.detach().requires_grad_(True), k, off)


@TYPES
def test_serving_steps(dtype):
    """As it is used: prompts normed, turned and written, then token after token in one captured step that writes and attends,
    replayed with growing lengths. Every step gives the eager call's bits, and what the oracle says of the values written;
    the prompt's attention over the cache is the one over the values read back."""
    h, hk, d, room = 4, 2, 64, 256
    prompts = [70, 1, 33]
    n, off = len(prompts), np.cumsum([0, *prompts])
    (qkv, qw, kw) = _normal(22, dtype, (off[-1], h + 2 * hk, d), (d,), (d,))
    pos = torch.cat([torch.arange(x) for x in prompts])[:, None].to(torch.int32).to(_dev())
    koff, fill = _int(np.arange(n + 1) * room), _int(prompts)
    q, k = norm_rotary_embed(qkv[:, :h], qkv[:, h:h + hk], qw, kw, pos, (32,))
    cache = new_cache4(n * room, hk, d, _dev())
    cache4_write(cache, k, qkv[:, h + hk:], _int(off), koff, fill)
    out = cache4_attention(q, cache, _int(off), koff, fill)
    back = cache4_read(cache, off[-1], _int(off), koff, fill, dtype=dtype)
    seqs = PA.sequences(off, koff.tolist(), prompts)
    _check(out, q, cache, seqs, SA.Shape(), False)
    packed = packed_attention(q, *back, _int(off))
    arrays = [_np(x) for x in (q, *back)]
    bound = SA.bounds(*arrays, np.zeros(arrays[0].shape), PA.sequences(off), HALF_STEP[dtype], SA.Shape())[0]
    assert (np.abs(_np(out) - _np(packed)) <= 2 * bound).all()

    new, place, step = torch.empty(n, h + 2 * hk, d, dtype=dtype, device=_dev()), fill.clone()[:, None], _int(range(n + 1))

    def work():
        tq, tk = norm_rotary_embed(new[:, :h], new[:, h:h + hk], qw, kw, place, (32,))
        cache4_write(cache, tk, new[:, h + hk:], step, koff, fill)
        return tq, cache4_attention(tq, cache, step, koff, fill, cap=10.0, window=64)

    fill += 1
    new.copy_(_normal(30, dtype, new.shape)[0])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        work()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        got = work()
    for i in range(4):
        new.copy_(_normal(30 + i, dtype, new.shape)[0])
        for x in got:
            x.fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        bytes_ = _bytes(cache)
        eager = work()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, eager))
        assert all((a == b).all() for a, b in zip(bytes_, _bytes(cache)))
        _check(got[1], got[0], cache, PA.sequences(range(n + 1), koff.tolist(), fill.tolist()), SA.Shape(cap=10.0, window=64), True)
        fill += 1
        place += 1


@TYPES
def test_two_at_once(dtype):
    """Calls on two streams over one cache, with workspaces of their own: the same bits each time."""
    lengths, fill, room, h, hk, d = SHAPES["tokens"]
    off, koff = np.cumsum([0, *lengths]), np.arange(len(fill) + 1) * room
    cache = _random_cache(23, koff[-1], hk, d)
    qs = _normal(24, dtype, *[(off[-1], h, d)] * 2)
    args = (_int(off), _int(koff), _int(fill))
    want = [cache4_attention(q, cache, *args) for q in qs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(4):
        got = []
        for q, s in zip(qs, streams):
            with torch.cuda.stream(s):
                got.append(cache4_attention(q, cache, *args))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
