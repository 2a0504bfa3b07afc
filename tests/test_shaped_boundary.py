"""Refusals of shaped scores, through the C ABI (validation runs before any HIP call) and the torch front-end, without
a GPU."""

from __future__ import annotations

import ctypes
import inspect

import pytest
import torch

from rfdetr_jax_amd import _native, packed_attention
from rfdetr_jax_amd.packed_attention import _Shape

PTR, ODD = ctypes.c_void_p(1 << 20), (1 << 20) + 2
INVALID, UNSUPPORTED = _native.ERR_INVALID_ARGUMENT, _native.ERR_UNSUPPORTED


def _call(direction, shape, causal=1, ws=None, ws_bytes=0, s=4, d=64):
    lib = _native.lib()
    strides = (ctypes.c_int64 * 16)(*([256, 64] * 8))
    dims = (1, 4, s, 4, 2, d)
    tail = (*dims, strides, causal, 0.125, None if shape is None else ctypes.byref(shape), ws, ws_bytes, None)
    if direction == "fwd":
        rc = lib.msda_packed_attention_shaped_fwd(PTR, PTR, PTR, 1, PTR, None, PTR, PTR, PTR, None, *tail)
    else:
        rc = lib.msda_packed_attention_shaped_bwd(PTR, PTR, PTR, PTR, None, PTR, PTR, PTR, 1, PTR, PTR, PTR, PTR, PTR, None, *tail)
    return rc, lib.msda_last_error().decode()


@pytest.mark.parametrize("direction", ["fwd", "bwd"])
@pytest.mark.parametrize("shape, causal, text", [
    (_native.ScoreShape(-1.0, 0, None, None), 1, "cap"), (_native.ScoreShape(float("nan"), 0, None, None), 1, "cap"),
    (_native.ScoreShape(2.0 ** -33, 0, None, None), 1, "cap"), (_native.ScoreShape(float("inf"), 0, None, None), 1, "cap"),
    (_native.ScoreShape(0.0, -1, None, None), 1, "window"), (_native.ScoreShape(0.0, 0, None, 1 << 20), 0, "causal"),
    (_native.ScoreShape(0.0, 0, ODD, None), 1, "4 bytes"), (_native.ScoreShape(0.0, 0, None, ODD), 1, "4 bytes"),
])
def test_c_refusals(direction, shape, causal, text):
    rc, msg = _call(direction, shape, causal)
    assert rc == INVALID and text in msg, (rc, msg)


def test_what_the_plain_calls_refuse():
    shape = _native.ScoreShape(30.0, 0, None, None)
    for direction in ("fwd", "bwd"):
        rc, msg = _call(direction, shape, d=60)
        assert rc == UNSUPPORTED and "head_dim" in msg
    # few rows over many keys: the forward needs a workspace
    rc, msg = _call("fwd", shape, s=100000)
    assert rc == INVALID and "workspace" in msg


def test_workspaces():
    lib = _native.lib()
    dims = (1, 64, 64, 64 * 8192, 32, 8, 128)
    plain = lib.msda_packed_attention_fwd_workspace_size(*dims)
    assert lib.msda_packed_attention_shaped_fwd_workspace_size(*dims, 0) == plain > 0
    assert 0 < lib.msda_packed_attention_shaped_fwd_workspace_size(*dims, 1024) < plain
    assert lib.msda_packed_attention_shaped_fwd_workspace_size(*dims, 64) == 0  # nothing to share
    train = (1, 2, 20000, 20000, 16, 4, 128)
    assert lib.msda_packed_attention_shaped_bwd_workspace_size(*train, 0) == lib.msda_packed_attention_bwd_workspace_size(*train) > 0
    assert lib.msda_packed_attention_shaped_bwd_workspace_size(*train, 128) == 0
    for name in ("fwd", "bwd"):
        assert getattr(lib, f"msda_packed_attention_shaped_{name}_workspace_size")(*train, -1) == INVALID
    # few tiles of queries: parts of dq, of 4 chunks of keys each at least, and each row's number of them
    few = (1, 1, 256, 256 * 16, 2, 1, 64)
    parts = lib.msda_packed_attention_shaped_bwd_workspace_size(*few, 0) - lib.msda_packed_attention_bwd_workspace_size(*few)
    assert parts == (8 * 64 + 1) * 256 * 2 * 4
    assert lib.msda_packed_attention_shaped_bwd_workspace_size(1, 1, 256, 448, 2, 1, 64, 0) == lib.msda_packed_attention_bwd_workspace_size(1, 1, 256, 448, 2, 1, 64)


CPU = torch.device("cpu")


@pytest.mark.parametrize("kw, error, text", [
    (dict(cap=0.0), ValueError, "cap"), (dict(cap=-3.0), ValueError, "cap"), (dict(cap=float("nan")), ValueError, "cap"),
    (dict(cap=2.0 ** 33), ValueError, "cap"), (dict(window=0), ValueError, "window"), (dict(window=1 << 31), ValueError, "window"),
    (dict(window=2.5), ValueError, "window"), (dict(slopes=torch.zeros(4, dtype=torch.bfloat16)), TypeError, "float32"),
    (dict(slopes=torch.zeros(3)), ValueError, r"\[4\]"), (dict(slopes=torch.zeros(4, requires_grad=True)), ValueError, "gradient"),
    (dict(slopes=torch.zeros(4, device="meta")), ValueError, "meta"), (dict(prefix_lengths=torch.zeros(2)), TypeError, "int32"),
    (dict(prefix_lengths=torch.zeros(3, dtype=torch.int32)), ValueError, r"\[2\]"),
    (dict(prefix_lengths=torch.zeros(2, dtype=torch.int32), causal=False), ValueError, "causal"),
])
def test_front_end_refusals(kw, error, text):
    args = dict(cap=None, slopes=None, window=None, prefix_lengths=None, causal=True)
    args.update(kw)
    with pytest.raises(error, match=text):
        _Shape(**args, heads=4, sequences=2, device=CPU)


def test_options_are_named_and_tensors_must_be_on_a_gpu():
    kinds = inspect.signature(packed_attention).parameters
    assert all(kinds[n].kind is inspect.Parameter.KEYWORD_ONLY and kinds[n].default is None for n in ("cap", "slopes", "window", "prefix_lengths"))
    q = torch.zeros(4, 2, 32)
    with pytest.raises(RuntimeError, match="no CPU path"):
        packed_attention(q, q, q, torch.tensor([0, 4], dtype=torch.int32), cap=30.0)
