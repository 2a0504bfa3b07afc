"""The oracle of the norms with rotary positions, against torch's float64 autograd and central differences, and planted
mistakes; the refusals of the C ABI and the front-end. Without a GPU."""

from __future__ import annotations

import ctypes

import numpy as np
import pytest
import torch

from oracle import norm_rotary_ref as NR
from rfdetr_jax_amd import _native, norm_rotary_embed

SECTIONS, EPS = (3, 2), 1e-3


def _arrays(seed=0):
    r = np.random.default_rng(seed)
    return r.standard_normal((5, 3, 14)), 1 + 0.3 * r.standard_normal(14), r.standard_normal((5, 3, 14)), r.integers(0, 50, (5, 2))


def _torch(x, w, dy, pos, interleaved, shared):
    x, w = (torch.tensor(t, requires_grad=True) for t in (x, w))
    n, columns = sum(SECTIONS), []
    for a, count in enumerate(SECTIONS):
        for j in range(count):
            e = len(columns) / n if shared else j / count
            columns.append(torch.tensor(pos[:, a], dtype=torch.float64) * 10000.0 ** -e)
    angle = torch.stack(columns, -1)[:, None]
    y = x / (x.pow(2).mean(-1, keepdim=True) + EPS).sqrt() * w
    a, b = (y[..., 0:2 * n:2], y[..., 1:2 * n:2]) if interleaved else (y[..., :n], y[..., n:2 * n])
    u, v = a * angle.cos() - b * angle.sin(), a * angle.sin() + b * angle.cos()
    y = torch.cat([torch.stack([u, v], -1).flatten(-2) if interleaved else torch.cat([u, v], -1), y[..., 2 * n:]], -1)
    return [t.detach().numpy() for t in (y, *torch.autograd.grad(y, (x, w), torch.tensor(dy)))]


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("shared", [False, True])
def test_against_autograd(interleaved, shared):
    x, w, dy, pos = _arrays()
    kw = dict(interleaved=interleaved, shared=shared)
    got = [NR.forward(x, w, pos, SECTIONS, EPS, **kw), *NR.backward(x, w, dy, pos, SECTIONS, EPS, **kw)]
    for a, b in zip(got, _torch(x, w, dy, pos, interleaved, shared)):
        np.testing.assert_allclose(a, b, rtol=0, atol=1e-12)
    ones = NR.backward(x, None, dy, pos, SECTIONS, EPS, **kw)
    for a, b in zip(ones, _torch(x, np.ones(14), dy, pos, interleaved, shared)[1:]):
        np.testing.assert_allclose(a, b, rtol=0, atol=1e-12)


def test_against_differences():
    x, w, dy, pos = _arrays(1)
    dx, dw = NR.backward(x, w, dy, pos, SECTIONS, EPS)
    r = np.random.default_rng(2)
    for i, grad in ((0, dx), (1, dw)):
        way, h, ends = r.standard_normal((x, w)[i].shape), 1e-6, []
        for sign in (1, -1):
            moved = [x, w]
            moved[i] = moved[i] + sign * h * way
            ends.append((NR.forward(*moved, pos, SECTIONS, EPS) * dy).sum())
        assert abs((ends[0] - ends[1]) / (2 * h) - (grad * way).sum()) < 1e-7


def test_planted_mistakes_leave_the_bounds():
    x, w, dy, pos = _arrays(3)
    want = [NR.forward(x, w, pos, SECTIONS, EPS), *NR.backward(x, w, dy, pos, SECTIONS, EPS)]
    bound = [NR.forward_bound(x, w, pos, SECTIONS, EPS, 2.0 ** -8), *NR.backward_bounds(x, w, dy, pos, SECTIONS, EPS, 2.0 ** -8, 2.0 ** -8)]
    r = 1 / np.sqrt((x * x).mean(-1, keepdims=True) + EPS)
    g = NR._turn(dy, pos, SECTIONS, {}, -1.0)
    wrong = [
        NR._turn(x * r, pos, SECTIONS, {}) * w,                       # the weight behind the rotation
        r * g * w,                                                    # the root as a constant
        (NR._turn(dy, pos, SECTIONS, {}) * x * r).sum((0, 1)),        # the cotangent turned the other way
    ]
    for a, b, c in zip(wrong, want, bound):
        assert (np.abs(a - b) > c).any()


PTR = ctypes.c_void_p(1 << 20)
ODD = ctypes.c_void_p((1 << 20) + 2)
INVALID, UNSUPPORTED = _native.ERR_INVALID_ARGUMENT, _native.ERR_UNSUPPORTED


def _call(direction, **kw):
    a = dict(q=PTR, y=PTR, k=PTR, ky=PTR, dtype=0, w=PTR, wt=0, pos=PTR, pt=0, t=4, h=4, hk=2, d=32, strides=None, ps=(2, 1), sections=(8, 8), axes=None,
             base=1e4, eps=1e-6, gw=PTR, ws=PTR, ws_bytes=1 << 20)
    a.update(kw)
    lib = _native.lib()
    n = 8 if direction == "fwd" else 12
    strides = (ctypes.c_int64 * n)(*([64, 32] * (n // 2) if a["strides"] is None else a["strides"] * (n // 2)))
    sections = None if a["sections"] is None else (ctypes.c_int32 * len(a["sections"]))(*a["sections"])
    axes = a["axes"] if a["axes"] is not None else len(a["sections"] or ())
    tail = (a["pos"], a["pt"], a["t"], a["h"], a["hk"], a["d"], strides, (ctypes.c_int64 * 2)(*a["ps"]), sections, axes, a["base"], 0, 0, a["eps"])
    if direction == "fwd":
        rc = lib.msda_norm_rotary_fwd(a["q"], a["y"], a["k"], a["ky"], a["dtype"], a["w"], a["w"], a["wt"], *tail, None)
    else:
        rc = lib.msda_norm_rotary_bwd(a["q"], a["y"], a["y"], a["k"], a["ky"], a["ky"], a["dtype"], a["w"], a["w"], a["gw"], a["gw"], a["wt"], *tail,
                                      a["ws"], a["ws_bytes"], None)
    return rc, lib.msda_last_error().decode()


@pytest.mark.parametrize("direction", ["fwd", "bwd"])
@pytest.mark.parametrize("change, code, text", [
    ({"dtype": 2}, UNSUPPORTED, "dtype"), ({"wt": 2}, UNSUPPORTED, "weight type"), ({"pt": 3}, UNSUPPORTED, "position type"), ({"t": -1}, INVALID, "negative"),
    ({"h": -1}, INVALID, "negative"), ({"d": 33}, UNSUPPORTED, "head_dim"), ({"d": 258}, UNSUPPORTED, "head_dim"), ({"d": 0}, UNSUPPORTED, "head_dim"),
    ({"h": 1 << 16}, UNSUPPORTED, "heads"), ({"sections": None, "axes": 1}, INVALID, "sections"), ({"axes": 0}, UNSUPPORTED, "axes"),
    ({"sections": (1,) * 9}, UNSUPPORTED, "axes"), ({"sections": (8, 0)}, INVALID, "section"), ({"sections": (8, 9)}, INVALID, "pairs"),
    ({"base": 0.0}, INVALID, "base"), ({"base": float("inf")}, INVALID, "base"), ({"eps": 0.0}, INVALID, "eps"), ({"eps": -1e-6}, INVALID, "eps"),
    ({"eps": float("nan")}, INVALID, "eps"), ({"eps": 1e-40}, INVALID, "eps"), ({"strides": [-64, 32]}, INVALID, "stride"), ({"ps": (-2, 1)}, INVALID, "stride"),
    ({"pos": None}, INVALID, "NULL"), ({"q": None}, INVALID, "NULL"), ({"ky": None}, INVALID, "NULL"), ({"q": ODD}, INVALID, "aligned"),
    ({"w": ODD}, INVALID, "aligned"), ({"pos": ODD}, INVALID, "aligned"),
])
def test_refusals(direction, change, code, text):
    rc, msg = _call(direction, **change)
    assert rc == code and text in msg, (rc, msg)


def test_workspace():
    lib = _native.lib()
    assert lib.msda_norm_rotary_bwd_workspace_size(4, 32) == 4 * 2 * 32 * 4
    assert lib.msda_norm_rotary_bwd_workspace_size(10 ** 8, 256) == 1024 * 2 * 256 * 4
    assert lib.msda_norm_rotary_bwd_workspace_size(-1, 32) == INVALID and lib.msda_norm_rotary_bwd_workspace_size(4, 7) == UNSUPPORTED
    for change in ({"ws": None}, {"ws_bytes": 100}, {"ws": ODD}):
        rc, msg = _call("bwd", **change)
        assert rc == INVALID and "workspace" in msg


def test_front_end_refuses_cpu_tensors():
    x = torch.zeros(4, 2, 32)
    with pytest.raises(RuntimeError, match="no CPU path"):
        norm_rotary_embed(x, x, None, None, torch.zeros(4, 1, dtype=torch.int32), (16,))
