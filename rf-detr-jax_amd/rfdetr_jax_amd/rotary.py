"""Rotary positions on several axes, on MI355X.

:func:`rotary_embed` turns the channel pairs of queries and keys by angles that grow with the token's
position on each axis (time, height and width of a video, rows and columns of an image, the one axis of a
text). Both tensors take one launch of ``msda_rotary``, and so do their gradients. There is no CPU path.
No counterpart in the reference.
"""

from __future__ import annotations

import ctypes

import torch
from torch.autograd.function import once_differentiable

from . import _native

_DTYPES = {torch.float32: _native.DTYPE_F32, torch.bfloat16: _native.DTYPE_BF16}
_POSITIONS = {torch.int32: _native.POSITION_I32, torch.int64: _native.POSITION_I64, torch.float32: _native.POSITION_F32}


def _ptr(t):
    return None if t is None else ctypes.c_void_p(t.data_ptr())


def _rows(t):
    """``[..., heads, D]`` as ``[T, heads, D]`` with contiguous channels (a view where there is one)."""
    t = t.flatten(0, -3) if t.dim() > 3 else t[None] if t.dim() == 2 else t
    return t if t.stride(-1) == 1 else t.contiguous()


def _rotate(q, k, positions, plan, inverse):
    """``(q', k')`` of ``[T, heads, D]`` tensors, contiguous; k may be None."""
    sections, base, shared, interleaved = plan
    outs = [None if t is None else torch.empty(t.shape, dtype=t.dtype, device=t.device) for t in (q, k)]
    flat = []
    for t in (q, outs[0], k, outs[1]):
        flat += [0, 0] if t is None else [t.stride(0), t.stride(1)]
    strides = (ctypes.c_int64 * 8)(*flat)
    where = (ctypes.c_int64 * 2)(positions.stride(0), positions.stride(1))
    pairs = (ctypes.c_int32 * len(sections))(*sections)
    with torch.cuda.device(q.device):
        rc = _native.lib().msda_rotary(_ptr(q), _ptr(outs[0]), _ptr(k), _ptr(outs[1]), _DTYPES[q.dtype], _ptr(positions),
                                       _POSITIONS[positions.dtype], q.shape[0], q.shape[1], 0 if k is None else k.shape[1], q.shape[2], strides,
                                       where, pairs, len(sections), base, int(shared), int(interleaved), int(inverse),
                                       ctypes.c_void_p(torch.cuda.current_stream(q.device).cuda_stream))
    _native.check(rc)
    return outs


class _Rotary(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, positions, plan):
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(positions)
        ctx.plan = plan
        outs = _rotate(_rows(q), None if k is None else _rows(k), positions, plan, False)
        if k is None:
            return outs[0].view(q.shape)
        return outs[0].view(q.shape), outs[1].view(k.shape)

    @staticmethod
    @once_differentiable
    def backward(ctx, *grads):
        (positions,) = ctx.saved_tensors
        shapes = [None if g is None else g.shape for g in grads]
        rows = [None if g is None else _rows(g) for g in grads]
        if len(rows) == 1:
            rows.append(None)
        outs = [None, None]
        if rows[0] is None and rows[1] is not None:  # one tensor is enough
            outs[1] = _rotate(rows[1], None, positions, ctx.plan, True)[0]
        elif rows[0] is not None:
            outs = _rotate(rows[0], rows[1], positions, ctx.plan, True)
        outs = [None if o is None else o.view(s) for o, s in zip(outs, [*shapes, None])]
        return outs[0], outs[1], None, None


def rotary_embed(q, k, positions, sections, base=10000.0, shared_frequencies=False, interleaved=False):
    """Rotates ``q`` and ``k`` by their tokens' positions: ``(q', k')``, or ``q'`` when ``k`` is None.

    Args:
        q: ``[..., H, D]`` float32 or bfloat16, ``D`` even, at most 256.
        k: ``[..., Hk, D]`` with the same leading shape and type, or None.
        positions: ``[..., A]`` int32, int64 or float32 on the same GPU (any strides): the position of each
            token on each of ``A <= 8`` axes. Far positions keep their precision (angles are formed in float64).
        sections: the number of channel pairs of each axis, in order; ``n`` is their sum, ``2 n <= D``. Channels
            from ``2 n`` on pass unchanged.
        base: pair ``i``, the ``j``-th of axis ``a``, turns by ``position_a * base ** -e``.
        shared_frequencies: ``e = i / n``, one falling sequence over all axes; False: ``e = j / sections[a]``,
            each axis its own.
        interleaved: pair ``i`` is the channels ``(2 i, 2 i + 1)``; False: ``(i, i + n)``.

    Differentiable in ``q`` and ``k`` (the rotation back), not in ``positions``, which get no gradient. Products are float32, rounded once.

    Raises:
        ValueError: shapes, devices or sizes that do not fit.
        TypeError: types other than the above.
        RuntimeError: tensors that are not on a GPU.
    """
    sections = tuple(int(s) for s in sections)
    out = _native.binding().rotary(q, k, positions, sections, base, bool(shared_frequencies), bool(interleaved))
    if out is not None:
        return out
    for name, t in (("q", q), ("k", k)):
        if t is None and name == "k":
            continue
        if t.device.type != "cuda":
            raise RuntimeError(f"tensor on {t.device}; the HIP kernels need GPU tensors (there is no CPU path)")
        if t.dtype not in _DTYPES:
            raise TypeError(f"{name} dtype {t.dtype} is not supported (float32 or bfloat16)")
        if t.dim() < 2:
            raise ValueError(f"{name} must be [..., heads, D], got {tuple(t.shape)}")
        if t.numel() >= (1 << 31) * max(t.shape[-1] * t.shape[-2], 1):
            raise ValueError(f"{name} holds too many tokens: {tuple(t.shape)}")
    if k is not None and (k.dtype != q.dtype or k.device != q.device):
        raise TypeError(f"q and k must be of one type and on one device, got {q.dtype} on {q.device} and {k.dtype} on {k.device}")
    if k is not None and (k.shape[:-2] != q.shape[:-2] or k.shape[-1] != q.shape[-1]):
        raise ValueError(f"q [..., H, D] and k [..., Hk, D] expected, got {tuple(q.shape)} and {tuple(k.shape)}")
    if positions.dtype not in _POSITIONS:
        raise TypeError(f"positions must be int32, int64 or float32, got {positions.dtype}")
    if positions.device != q.device:
        raise ValueError(f"positions are on {positions.device}, the queries on {q.device}")
    if not 1 <= len(sections) <= 8 or min(sections) < 1:
        raise ValueError(f"sections must be 1 to 8 numbers of pairs, got {sections}")
    if tuple(positions.shape) != (*q.shape[:-2], len(sections)):
        raise ValueError(f"positions must be {[*q.shape[:-2], len(sections)]}, got {tuple(positions.shape)}")
    if q.shape[-1] % 2 or q.shape[-1] > 256 or 2 * sum(sections) > q.shape[-1]:
        raise ValueError(f"D = {q.shape[-1]} must be even, at most 256, and hold {sum(sections)} pairs")
    base = float(base)
    if not 0.0 < base < float("inf"):
        raise ValueError(f"base must be positive and finite, got {base}")
    return _Rotary.apply(q, k, positions.flatten(0, -2) if positions.dim() > 1 else positions[None], (sections, base, bool(shared_frequencies), bool(interleaved)))
