"""Attention over a cache in 4 bits on an MI355X: places past 2^24, blocks that are not finite wherever the parts of a
call fall. Tolerances are those of shaped_attention_ref's ``bounds``."""

from __future__ import annotations

import sys

import numpy as np
import pytest
import torch

from oracle import cache4_ref as C4
from oracle import shaped_attention_ref as SA
from rfdetr_jax_amd import Cache4, cache4_attention, packed_attention

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


def _random_cache(seed, rows, hk, d):
    r = np.random.default_rng(seed)
    blocks = (d + 31) // 32
    out = []
    for _ in range(2):
        codes = r.integers(0, 16, (hk, rows, 32 * blocks)).astype(np.uint8)
        codes[..., d:] = 0
        out += [codes[..., 0::2] | codes[..., 1::2] << 4, (126 + r.integers(-2, 2, (hk, rows, blocks))).astype(np.uint8)]
    return Cache4(*(torch.from_numpy(x).to(_dev()) for x in out), d)


def _held(cache):
    b = [t.cpu().numpy() for t in cache[:4]]
    return [C4.decode(b[i], b[i + 1], cache.head_dim).transpose(1, 0, 2) for i in (0, 2)]


def _check(out, q, cache, seqs, shape):
    arrays, u = [_np(q), *_held(cache)], HALF_STEP[q.dtype]
    want = SA.attention(*arrays, seqs, shape)
    bound = SA.bounds(*arrays, np.zeros(arrays[0].shape), seqs, u, shape)[0]
    got = _np(out)
    assert np.isfinite(got).all()
    over = np.abs(got - want) - bound
    at = np.unravel_index(np.argmax(over), over.shape)
    assert over[at] <= 0, f"off by {abs(got[at] - want[at]):.3e} at {at}, {bound[at]:.3e} allowed"


@TYPES
@pytest.mark.parametrize("n", [1, 3, 50], ids=["token", "tokens", "chunk"])  # 50: rows in tiles
def test_distances_past_2_to_the_24(n, dtype):
    """The newest queries of a sequence of more than 2^24 keys, inside a window; unseen blocks are not finite."""
    m, h, d, window, tail = (1 << 24) + 301, 2, 40, 70, 256
    sys.stderr.write(f"[gpu] cache in 4 bits, distances past 2^24, {n} tokens {dtype}\n")
    small = _random_cache(1, tail, 1, d)
    cache = Cache4(*(torch.cat([torch.full((1, m - tail, t.shape[2]), 255, dtype=torch.uint8, device=_dev()), t], 1) for t in small[:4]), d)
    (q,) = _normal(2, dtype, (n, h, d))
    slopes = torch.tensor([1.0, 0.37], device=_dev())
    for kw in (dict(), dict(cap=3.0), dict(causal=False)):
        out = cache4_attention(q, cache, _int([0, n]), _int([0, m]), slopes=slopes, window=window, **kw)
        _check(out, q, small, [(0, n, 0, tail)], SA.Shape(kw.get("causal", True), None, kw.get("cap"), _np(slopes), window))


@TYPES
@pytest.mark.parametrize("n", [1, 3, 50], ids=["token", "tokens", "chunk"])
def test_a_bad_value_of_a_part_that_weighs_nothing(n, dtype):
    """Slopes so steep that the first part of the keys weighs 0 beside the last: a block of its values that is not finite
    makes the rows that see it NaN all the same, in its channels alone."""
    m, h, hk, d = 5000, 4, 2, 64
    cache = _random_cache(3, m, hk, d)
    (q,) = _normal(4, dtype, (n, h, d))
    args = (_int([0, n]), _int([0, m]))
    slopes = torch.full((h,), 0.5, device=_dev())
    want = cache4_attention(q, cache, *args, slopes=slopes)
    _check(want, q, cache, [(0, n, 0, m)], SA.Shape(slopes=_np(slopes)))
    for key in (10, 2600):
        bad = Cache4(*(t.clone() for t in cache[:4]), d)
        bad.value_scales[1, key, 1] = 255
        got = cache4_attention(q, bad, *args, slopes=slopes)
        assert torch.isnan(got[:, 2:, 32:]).all()
        assert torch.equal(got[:, 2:, :32], want[:, 2:, :32]) and torch.equal(got[:, :2], want[:, :2])


@TYPES
@pytest.mark.parametrize("d", [72, 96])
def test_what_an_earlier_kernel_left_does_not_matter(d, dtype):
    """Rows of 72 to 96 channels lie 128 apart in LDS. A kernel before this one that left NaN everywhere there changes neither
    the results nor, by more than the clock's noise, the time (unwritten channels once took ten times as long)."""
    n, m, h, hk = 200, 6000, 8, 8
    cache = _random_cache(5, m, hk, d)
    (q,) = _normal(6, dtype, (n, h, d))
    zeros = torch.zeros(4096, 8, 128, device=_dev())
    places, kw = (_int([0, n]), _int([0, m])), dict(window=4000)

    def call(left):
        keys = torch.full((4096, 8, 128), left, dtype=torch.int32, device=_dev()).view(torch.float32)
        times = []
        for _ in range(7):
            packed_attention(zeros, keys, keys, _int([0, 4096]), causal=False)
            start, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
            start.record()
            out = cache4_attention(q, cache, *places, **kw)
            end.record()
            torch.cuda.synchronize()
            times.append(start.elapsed_time(end))
        return out, sorted(times)[2]

    call(0)
    (want, clean), (got, odd) = call(0), call(0x7FFFFFFF)
    _check(want, q, cache, [(0, n, 0, m)], SA.Shape(window=4000))
    assert torch.equal(got, want)
    assert odd < 3 * clean, f"{1e3 * odd:.0f} us behind NaN, {1e3 * clean:.0f} behind zeros"
