"""Refusals of the packed attention and the rotary positions, through the C ABI (validation runs before any HIP
call) and the torch front-end, without a GPU."""

from __future__ import annotations

import ctypes

import pytest
import torch

from rfdetr_jax_amd import _native, packed_attention, rotary_embed

PTR = ctypes.c_void_p(1 << 20)
ODD = ctypes.c_void_p((1 << 20) + 8)


def _i64(*v):
    return (ctypes.c_int64 * len(v))(*v)


def _attention(direction, **kw):
    a = dict(q=PTR, k=PTR, v=PTR, dtype=1, out=PTR, rest=None, stats=PTR, qo=PTR, ko=PTR, kl=None, n=1, t=4, s=4, h=4, hk=2, d=64, causal=1, scale=0.125,
             strides=None, ws=None, ws_bytes=0, go=PTR, gq=PTR, gk=PTR, gv=PTR)
    a.update(kw)
    lib = _native.lib()
    dims = (a["n"], a["t"], a["s"], a["h"], a["hk"], a["d"])
    strides = _i64(*([256, 64] * (4 if direction == "fwd" else 8))) if a["strides"] is None else a["strides"]
    if direction == "fwd":
        rc = lib.msda_packed_attention_fwd(a["q"], a["k"], a["v"], a["dtype"], a["out"], a["rest"], a["stats"], a["qo"], a["ko"], a["kl"], *dims, strides,
                                           a["causal"], a["scale"], a["ws"], a["ws_bytes"], None)
    else:
        rc = lib.msda_packed_attention_bwd(a["q"], a["k"], a["v"], a["out"], a["rest"], a["stats"], a["go"], a["dtype"], a["gq"], a["gk"], a["gv"], a["qo"],
                                           a["ko"], a["kl"], *dims, strides, a["causal"], a["scale"], a["ws"], a["ws_bytes"], None)
    return rc, lib.msda_last_error().decode()


INVALID, UNSUPPORTED = _native.ERR_INVALID_ARGUMENT, _native.ERR_UNSUPPORTED


@pytest.mark.parametrize("direction", ["fwd", "bwd"])
@pytest.mark.parametrize("change, code, text", [
    ({"dtype": 2}, UNSUPPORTED, "dtype"), ({"n": -1}, INVALID, "negative"), ({"t": -4}, INVALID, "negative"), ({"d": 60}, UNSUPPORTED, "head_dim"),
    ({"d": 136}, UNSUPPORTED, "head_dim"), ({"d": 0}, UNSUPPORTED, "head_dim"), ({"h": 5}, INVALID, "divide"), ({"hk": 0}, INVALID, "divide"),
    ({"h": 0}, INVALID, "divide"), ({"h": 0, "hk": 0}, INVALID, "divide"),
    ({"t": 2 ** 31 - 1}, UNSUPPORTED, "rows"), ({"s": 2 ** 31 - 1}, UNSUPPORTED, "rows"), ({"n": 2 ** 25}, UNSUPPORTED, "rows"),
    ({"scale": 0.0}, INVALID, "scale"), ({"scale": -1.0}, INVALID, "scale"), ({"scale": float("nan")}, INVALID, "scale"),
    ({"scale": float("inf")}, INVALID, "scale"), ({"q": None}, INVALID, "NULL"), ({"k": None}, INVALID, "NULL"), ({"out": None}, INVALID, "NULL"),
    ({"qo": None}, INVALID, "offsets"), ({"ko": None}, INVALID, "offsets"), ({"v": ODD}, INVALID, "16 bytes"), ({"stats": ODD}, INVALID, "16 bytes"),
    ({"kl": ctypes.c_void_p((1 << 20) + 2)}, INVALID, "4 bytes"), ({"strides": _i64(*([260, 64] * 8))}, INVALID, "stride"),
    ({"strides": _i64(*([-256, 64] * 8))}, INVALID, "stride"), ({"strides": _i64(*([56, 64] * 8))}, UNSUPPORTED, "apart"),
    ({"strides": _i64(*([1 << 22, 64] * 8))}, UNSUPPORTED, "apart"), ({"strides": _i64(*([256, 1 << 26] * 8))}, UNSUPPORTED, "apart"),
    ({"rest": ODD}, INVALID, "16 bytes"), ({"h": 130, "hk": 2}, UNSUPPORTED, "key head"), ({"scale": 2.0 ** -65}, INVALID, "scale"),
    ({"scale": 2.0 ** 65}, INVALID, "scale"),
])
def test_attention_refusals(direction, change, code, text):
    rc, msg = _attention(direction, **change)
    assert rc == code and text in msg, (rc, msg)


def test_attention_backward_pointers_and_workspace():
    assert _attention("bwd", go=None)[0] == INVALID and _attention("bwd", stats=None)[0] == INVALID
    assert _attention("bwd", gk=ODD)[0] == INVALID
    assert _attention("bwd", gq=None, gk=None, gv=None)[0] == 0  # nothing wanted, nothing launched
    assert _attention("fwd", t=0)[0] == 0 and _attention("bwd", t=0, s=0)[0] == 0
    size = _native.lib().msda_packed_attention_fwd_workspace_size
    assert size(1, 1, 4096, 4096, 32, 8, 128) == 0
    need = size(1, 1, 1, 100000, 8, 8, 128)  # one token: its keys are split
    assert need > 0 and need % 4 == 0
    assert size(1, 1, 1, 100000, 8, 3, 128) == INVALID and size(7, 1, 1, 1, 8, 8, 128) == UNSUPPORTED
    for ws, n in ((None, 0), (PTR, need - 1), (ODD, need)):
        rc, msg = _attention("fwd", t=1, s=100000, h=8, hk=8, d=128, strides=_i64(*([1024, 128] * 4)), ws=ws, ws_bytes=n)
        assert rc == INVALID and "workspace" in msg
    size = _native.lib().msda_packed_attention_bwd_workspace_size
    assert size(1, 16, 65536, 65536, 32, 8, 128) == 0
    need = size(1, 1, 4096, 4096, 16, 2, 64)  # 64 tiles of keys: several workgroups share one
    assert need > 0 and need % (2 * 4096 * 2 * 64 * 4) == 0
    big = dict(t=4096, s=4096, h=16, hk=2, strides=_i64(*([1024, 64] * 8)))
    for ws, n in ((None, 0), (PTR, need - 1), (ODD, need)):
        rc, msg = _attention("bwd", ws=ws, ws_bytes=n, **big)
        assert rc == INVALID and "workspace" in msg


def _rotary(**kw):
    a = dict(q=PTR, qy=PTR, k=PTR, ky=PTR, dtype=0, pos=PTR, pt=0, t=4, h=2, hk=1, d=32, strides=_i64(*([64, 32] * 4)), ps=_i64(2, 1),
             sections=(8, 8), axes=None, base=10000.0)
    a.update(kw)
    lib = _native.lib()
    sections = None if a["sections"] is None else (ctypes.c_int32 * len(a["sections"]))(*a["sections"])
    rc = lib.msda_rotary(a["q"], a["qy"], a["k"], a["ky"], a["dtype"], a["pos"], a["pt"], a["t"], a["h"], a["hk"], a["d"], a["strides"], a["ps"],
                         sections, len(a["sections"] or ()) if a["axes"] is None else a["axes"], a["base"], 0, 0, 0, None)
    return rc, lib.msda_last_error().decode()


@pytest.mark.parametrize("change, code, text", [
    ({"dtype": 3}, UNSUPPORTED, "dtype"), ({"pt": 3}, UNSUPPORTED, "position"), ({"pt": -1}, UNSUPPORTED, "position"), ({"t": -1}, INVALID, "negative"),
    ({"d": 31}, UNSUPPORTED, "head_dim"), ({"d": 258}, UNSUPPORTED, "head_dim"), ({"d": 0}, UNSUPPORTED, "head_dim"), ({"h": 70000}, UNSUPPORTED, "heads"),
    ({"axes": 0}, UNSUPPORTED, "axes"), ({"sections": (1,) * 9}, UNSUPPORTED, "axes"), ({"sections": None, "axes": 1}, INVALID, "NULL"),
    ({"sections": (8, 0)}, INVALID, "section"), ({"sections": (8, 9)}, INVALID, "fit"), ({"sections": (2 ** 31 - 1, 2 ** 31 - 1)}, INVALID, "fit"),
    ({"base": 0.0}, INVALID, "base"), ({"base": float("nan")}, INVALID, "base"), ({"base": float("inf")}, INVALID, "base"),
    ({"pos": None}, INVALID, "NULL"), ({"q": None}, INVALID, "NULL"), ({"ky": None}, INVALID, "NULL"),
    ({"q": ctypes.c_void_p((1 << 20) + 2)}, INVALID, "aligned"), ({"strides": _i64(*([-64, 32] * 4))}, INVALID, "stride"),
    ({"ps": _i64(-2, 1)}, INVALID, "stride"),
])
def test_rotary_refusals(change, code, text):
    rc, msg = _rotary(**change)
    assert rc == code and text in msg, (rc, msg)


def test_front_end_refuses_cpu_tensors_and_other_types():
    x = torch.zeros(4, 2, 32)
    off = torch.tensor([0, 4], dtype=torch.int32)
    with pytest.raises(RuntimeError, match="no CPU path"):
        packed_attention(x, x, x, off)
    with pytest.raises(RuntimeError, match="no CPU path"):
        rotary_embed(x, x, torch.zeros(4, 1, dtype=torch.int32), (16,))


def test_attention_backward_with_row_numbers_of_its_own():
    lib, strides = _native.lib(), _i64(*([256, 64] * 8))

    def call(numbers, **kw):
        a = dict(stats=PTR, go=PTR, gq=PTR, gk=PTR, gv=PTR, scale=0.125, d=64)
        a.update(kw)
        rc = lib.msda_packed_attention_bwd_const(PTR, PTR, PTR, PTR, None, a["stats"], numbers, a["go"], 1, a["gq"], a["gk"], a["gv"], PTR, PTR, None,
                                                 1, 4, 4, 4, 2, a["d"], strides, 1, a["scale"], None, 0, None)
        return rc, lib.msda_last_error().decode()

    for numbers, change, code, text in ((None, {}, INVALID, "NULL"), (None, {"gq": None, "gk": None}, INVALID, "NULL"), (ODD, {}, INVALID, "16 bytes"),
                                        (PTR, {"stats": None}, INVALID, "NULL"), (PTR, {"go": None}, INVALID, "NULL"), (PTR, {"scale": 0.0}, INVALID, "scale"),
                                        (PTR, {"d": 60}, UNSUPPORTED, "head_dim")):
        rc, msg = call(numbers, **change)
        assert rc == code and text in msg, (rc, msg)
    assert call(None, gq=None, gk=None, gv=None)[0] == 0


@pytest.mark.parametrize("direction", ["fwd", "bwd"])
def test_rows_on_top_of_each_other_are_refused(direction):
    """Strides of 0 stand for a tensor that is not there: a gradient that is not wanted."""
    tensors = 4 if direction == "fwd" else 8
    for i in range(tensors):
        strides = [256, 64] * tensors
        strides[2 * i:2 * i + 2] = [0, 0]
        rc, msg = _attention(direction, strides=_i64(*strides))
        assert rc == UNSUPPORTED and "apart" in msg, (i, rc, msg)
    if direction == "bwd":
        assert _attention(direction, strides=_i64(*([256, 64] * 5 + [0, 0] * 3)), gq=None, gk=None, gv=None)[0] == 0


def test_key_heads_whose_row_numbers_pass_31_bits_are_refused():
    """A tile's numbers lie up to 64 rows of all heads apart, 16 bytes each: 2^21 key heads head-major, whatever the group."""
    for hk, group in ((1 << 21, 1), (1 << 21, 2), (1 << 24, 1)):
        rc, msg = _attention("bwd", t=64, s=64, h=hk * group, hk=hk, d=8, strides=_i64(*([8, 512] * 8)))
        assert rc == UNSUPPORTED and "key heads" in msg, (rc, msg)
