"""The oracle of the cache in 4 bits, and the refusals of its C ABI and front-end. Without a GPU."""

from __future__ import annotations

import ctypes

import numpy as np
import pytest
import torch

from oracle import cache4_ref as C4
from rfdetr_jax_amd import Cache4, _native, cache4_attention, cache4_read, cache4_write, new_cache4


def test_values_that_the_codes_hold_come_back():
    r = np.random.default_rng(0)
    block = np.concatenate([C4.MAGNITUDES, -np.array(C4.MAGNITUDES), r.choice(C4.MAGNITUDES, 16)])
    for e in (-120, -60, -1, 0, 7, 125):
        x = block * 2.0 ** e
        codes, scales = C4.encode(x[None])
        assert scales[0, 0] == e + 127
        np.testing.assert_array_equal(C4.decode(codes, scales, 32)[0], x)


def test_ties_go_to_the_even_code_and_the_scale_is_the_least():
    x = np.zeros(32)
    x[:8] = [6, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0]
    codes, scales = C4.encode(x[None])
    assert list(C4.decode(codes, scales, 32)[0, :8]) == [6, 0, 1, 1, 2, 2, 4, 4]
    for top, want in ((7.0, 6.0), (7.0001, 8.0), (6.0, 6.0), (3.5, 3.0), (3.6, 4.0)):
        x = np.zeros(32)
        x[5] = -top
        codes, scales = C4.encode(x[None])
        assert C4.decode(codes, scales, 32)[0, 5] == -want


def test_edges():
    for x, want in ((np.zeros(40), np.zeros(40)), (np.full(40, 1e-45), np.zeros(40)), (np.full(40, 3e38), np.full(40, 6 * 2.0 ** 125))):
        codes, scales = C4.encode(x[None])
        assert codes.shape == (1, 32) and scales.shape == (1, 2)
        np.testing.assert_array_equal(C4.decode(codes, scales, 40)[0], want)
    x = np.ones(64)
    x[3], x[40] = np.inf, 2.0
    codes, scales = C4.encode(x[None])
    got = C4.decode(codes, scales, 64)[0]
    assert np.isnan(got[:32]).all() and got[40] == 2.0 and (got[41:] == 1.0).all()


def test_error_is_half_a_step():
    r = np.random.default_rng(1)
    x = r.standard_normal((50, 96)) * np.exp(r.standard_normal((50, 1)) * 5)
    codes, scales = C4.encode(x)
    got = C4.decode(codes, scales, 96)
    unit = np.repeat(2.0 ** (scales.astype(float) - 127), 32, -1)
    step = np.where(np.abs(x) / unit <= 2, 0.25, np.where(np.abs(x) / unit <= 4, 0.5, 1.0)) * unit
    assert (np.abs(got - x) <= step).all()


PTR, ODD = ctypes.c_void_p(1 << 20), ctypes.c_void_p((1 << 20) + 8)
INVALID, UNSUPPORTED = _native.ERR_INVALID_ARGUMENT, _native.ERR_UNSUPPORTED


def _call(what, **kw):
    a = dict(x=PTR, y=PTR, dtype=1, codes=PTR, scales=PTR, qo=PTR, ko=PTR, kl=None, n=1, t=4, s=64, h=4, hk=2, d=64, strides=(256, 64, 256, 64), causal=1, scale=0.125,
             shape=None, ws=None, ws_bytes=0)
    a.update(kw)
    lib = _native.lib()
    cache = (a["codes"], a["scales"], a["codes"], a["scales"])
    places = (a["qo"], a["ko"], a["kl"])
    strides = None if a["strides"] is None else (ctypes.c_int64 * 4)(*a["strides"])
    if what == "attention":
        shape = None if a["shape"] is None else ctypes.byref(a["shape"])
        rc = lib.msda_cache4_attention(a["x"], a["dtype"], a["y"], *cache, *places, a["n"], a["t"], a["s"], a["h"], a["hk"], a["d"], strides, a["causal"], a["scale"],
                                       shape, a["ws"], a["ws_bytes"], None)
    elif what == "write":
        rc = lib.msda_cache4_write(a["x"], a["y"], a["dtype"], *cache, *places, a["n"], a["t"], a["s"], a["hk"], a["d"], strides, None)
    else:
        rc = lib.msda_cache4_read(*cache, a["x"], a["y"], a["dtype"], *places, a["n"], a["t"], a["s"], a["hk"], a["d"], strides, None)
    return rc, lib.msda_last_error().decode()


@pytest.mark.parametrize("what", ["write", "read", "attention"])
@pytest.mark.parametrize("change, code, text", [
    ({"dtype": 2}, UNSUPPORTED, "dtype"), ({"n": -1}, INVALID, "negative"), ({"t": -4}, INVALID, "negative"), ({"s": -4}, INVALID, "negative"),
    ({"d": 60}, UNSUPPORTED, "head_dim"), ({"d": 136}, UNSUPPORTED, "head_dim"), ({"hk": 0}, INVALID, "divide"), ({"n": 1 << 24}, UNSUPPORTED, "many"),
    ({"t": 2 ** 31 - 1}, UNSUPPORTED, "rows"), ({"s": 2 ** 31 - 1}, UNSUPPORTED, "rows"), ({"hk": 1 << 16, "h": 1 << 16}, UNSUPPORTED, "many"),
    ({"strides": None}, INVALID, "strides"), ({"strides": (260, 64, 260, 64)}, INVALID, "stride"), ({"strides": (-256, 64, 256, 64)}, INVALID, "stride"),
    ({"qo": None}, INVALID, "offsets"), ({"ko": None}, INVALID, "offsets"), ({"kl": ctypes.c_void_p((1 << 20) + 2)}, INVALID, "4 bytes"),
    ({"codes": None}, INVALID, "NULL"), ({"scales": None}, INVALID, "NULL"), ({"codes": ODD}, INVALID, "16 bytes"), ({"x": None}, INVALID, "NULL"),
    ({"y": None}, INVALID, "NULL"), ({"y": ODD}, INVALID, "16 bytes"),
])
def test_c_refusals(what, change, code, text):
    rc, msg = _call(what, **change)
    assert rc == code and text in msg, (rc, msg)


@pytest.mark.parametrize("change, code, text", [
    ({"h": 5}, INVALID, "divide"), ({"h": 130}, UNSUPPORTED, "key head"), ({"scale": 0.0}, INVALID, "scale"), ({"scale": 2.0 ** 65}, INVALID, "scale"),
    ({"strides": (56, 64, 256, 64)}, UNSUPPORTED, "apart"), ({"shape": _native.ScoreShape(-1.0, 0, None, None)}, INVALID, "cap"),
    ({"shape": _native.ScoreShape(0.0, 0, None, 1 << 20), "causal": 0}, INVALID, "causal"), ({"s": 100000, "t": 1}, INVALID, "workspace"),
])
def test_attention_refusals(change, code, text):
    rc, msg = _call("attention", **change)
    assert rc == code and text in msg, (rc, msg)


def test_workspace():
    size = _native.lib().msda_cache4_attention_workspace_size
    assert size(1, 64, 64, 64 * 512, 32, 8, 128, 0) == 0
    assert size(1, 64, 64, 64 * 8192, 32, 8, 128, 0) > size(1, 64, 64, 64 * 8192, 32, 8, 128, 2048) > 0
    assert size(1, 1, 1, 1, 4, 2, 60, 0) == UNSUPPORTED and size(1, 1, 1, 1, 4, 2, 64, -1) == INVALID


def test_front_end_refusals():
    for kw in (dict(head_dim=60), dict(head_dim=136), dict(rows=-1), dict(kv_heads=0)):
        args = dict(rows=8, kv_heads=2, head_dim=64, device="cpu")
        args.update(kw)
        with pytest.raises(ValueError):
            new_cache4(**args)
    cache = new_cache4(8, 2, 40, "cpu")
    assert isinstance(cache, Cache4) and cache.rows == 8 and cache.kv_heads == 2
    assert [tuple(t.shape) for t in cache[:4]] == [(2, 8, 32), (2, 8, 2)] * 2
    x, off = torch.zeros(4, 2, 40), torch.tensor([0, 4], dtype=torch.int32)
    for call in (lambda: cache4_write(cache, x, x, off), lambda: cache4_read(cache, 4, off), lambda: cache4_attention(x, cache, off)):
        with pytest.raises(RuntimeError, match="no CPU path"):
            call()
    with pytest.raises(TypeError, match="dtype"):
        cache4_read(cache, 4, off, dtype=torch.float16)
    with pytest.raises(ValueError, match="tokens"):
        cache4_read(cache, -1, off)
    for empty in (Cache4(*(torch.empty(0, 8, n, dtype=torch.uint8) for n in (32, 2) * 2), 40), cache._replace(keys=cache.keys[0])):
        for call in (lambda: cache4_write(empty, x, x, off), lambda: cache4_attention(x, empty, off)):
            with pytest.raises(ValueError, match="at least one head"):
                call()


def test_scales_that_no_block_gets_are_not_finite():
    codes, scales = np.full((3, 16), 0x22, np.uint8), np.array([[252], [253], [255]], np.uint8)
    got = C4.decode(codes, scales, 32)
    assert (got[0] == 2.0 ** 125).all() and np.isnan(got[1:]).all()
