"""Calls of more workgroups than a launch takes (its threads are counted in 32 bits) are refused before any launch, so no
GPU is needed."""

from __future__ import annotations

import ctypes

import pytest

from rfdetr_jax_amd import _native

PTR = ctypes.c_void_p(1 << 20)


@pytest.mark.parametrize("what", ["write", "read"])
@pytest.mark.parametrize("tokens, heads, dim", [(1 << 24, 8, 128), (1 << 30, 1, 8)])
def test_rows_of_a_cache(what, tokens, heads, dim):
    lib, places = _native.lib(), (PTR, PTR, None, 1, tokens, 64, heads, dim)
    strides = (ctypes.c_int64 * 4)(heads * dim, dim, heads * dim, dim)
    if what == "write":
        rc = lib.msda_cache4_write(PTR, PTR, 1, PTR, PTR, PTR, PTR, *places, strides, None)
    else:
        rc = lib.msda_cache4_read(PTR, PTR, PTR, PTR, PTR, PTR, 1, *places, strides, None)
    assert rc == _native.ERR_UNSUPPORTED and "too many workgroups" in lib.msda_last_error().decode()


@pytest.mark.parametrize("dim", [8, 6])  # rows on 16-byte boundaries, and others
def test_norms_of_many_tokens(dim):
    lib = _native.lib()
    strides, sections = (ctypes.c_int64 * 8)(*([dim, dim] * 4)), (ctypes.c_int32 * 1)(dim // 2)
    rc = lib.msda_norm_rotary_fwd(PTR, PTR, None, None, 0, None, None, 0, PTR, 0, 1 << 27, 1, 0, dim, strides, (ctypes.c_int64 * 2)(1, 1), sections, 1, 1e4, 0, 0,
                                  1e-6, None)
    assert rc == _native.ERR_UNSUPPORTED and "too many tokens" in lib.msda_last_error().decode()
