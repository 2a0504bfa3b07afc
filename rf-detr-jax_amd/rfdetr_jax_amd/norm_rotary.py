"""Norms of queries and keys for each head, with the rotary positions in the same pass, on MI355X.

:func:`norm_rotary_embed` divides every head of every token by the root of its mean square, multiplies it with a weight
and turns it by the token's positions as :func:`~rfdetr_jax_amd.rotary_embed` does: one read and one write of the rows
where a norm and a rotation apart take two each. Queries and keys take one launch of ``msda_norm_rotary_fwd``, and their
gradients, the weights' included, one of ``msda_norm_rotary_bwd``. There is no CPU path. No counterpart in the reference.
"""

from __future__ import annotations

import ctypes

import torch
from torch.autograd.function import once_differentiable

from . import _native
from .rotary import _DTYPES, _POSITIONS, _ptr, _rows


def _arguments(q, k, positions, tensors, plan):
    """The arguments behind the tensors that both directions share, and the strides of ``tensors``."""
    sections, base, shared, interleaved, eps = plan
    flat = []
    for t in tensors:
        flat += [0, 0] if t is None else [t.stride(0), t.stride(1)]
    like = q if q is not None else k
    return (_ptr(positions), _POSITIONS[positions.dtype], like.shape[0], 0 if q is None else q.shape[1], 0 if k is None else k.shape[1], like.shape[2],
            (ctypes.c_int64 * len(flat))(*flat), (ctypes.c_int64 * 2)(positions.stride(0), positions.stride(1)),
            (ctypes.c_int32 * len(sections))(*sections), len(sections), base, int(shared), int(interleaved), eps)


def _weight_type(*weights):
    return next((_DTYPES[w.dtype] for w in weights if w is not None), _native.DTYPE_F32)


def _forward(q, k, q_weight, k_weight, positions, plan):
    outs = [None if t is None else torch.empty(t.shape, dtype=t.dtype, device=t.device) for t in (q, k)]
    with torch.cuda.device(q.device):
        rc = _native.lib().msda_norm_rotary_fwd(_ptr(q), _ptr(outs[0]), _ptr(k), _ptr(outs[1]), _DTYPES[q.dtype], _ptr(q_weight), _ptr(k_weight),
                                                _weight_type(q_weight, k_weight), *_arguments(q, k, positions, (q, outs[0], k, outs[1]), plan),
                                                ctypes.c_void_p(torch.cuda.current_stream(q.device).cuda_stream))
    _native.check(rc)
    return outs


def _backward(q, gq, k, gk, q_weight, k_weight, positions, plan, needs):
    """Gradients of (q, k, q_weight, k_weight) where ``needs`` says so; q or k (and its cotangent) may be None."""
    like = q if q is not None else k
    grads = [torch.empty(t.shape, dtype=t.dtype, device=t.device) if need and t is not None else None for t, need in zip((q, k), needs)]
    sums = [torch.empty_like(w) if need and w is not None else None for w, need in zip((q_weight, k_weight), needs[2:])]
    with torch.cuda.device(like.device):
        lib, ws, nbytes = _native.lib(), None, 0
        if any(s is not None for s in sums):
            nbytes = lib.msda_norm_rotary_bwd_workspace_size(like.shape[0], like.shape[2])
            _native.check(min(nbytes, 0))
            ws = _native.workspace(nbytes, like.device)
        rc = lib.msda_norm_rotary_bwd(_ptr(q), _ptr(gq), _ptr(grads[0]), _ptr(k), _ptr(gk), _ptr(grads[1]), _DTYPES[like.dtype], _ptr(q_weight),
                                      _ptr(k_weight), _ptr(sums[0]), _ptr(sums[1]), _weight_type(q_weight, k_weight),
                                      *_arguments(q, k, positions, (q, gq, grads[0], k, gk, grads[1]), plan), _ptr(ws), nbytes,
                                      ctypes.c_void_p(torch.cuda.current_stream(like.device).cuda_stream))
    _native.check(rc)
    return (*grads, *sums)


class _NormRotary(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, q_weight, k_weight, positions, plan):
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(q, k, q_weight, k_weight, positions)
        ctx.plan = plan
        ctx.types = [None if w is None else w.dtype for w in (q, k, q_weight, k_weight)]
        weights = [None if w is None else w.contiguous() for w in (q_weight, k_weight)]
        outs = _forward(_rows(q), None if k is None else _rows(k), *weights, positions, plan)
        if k is None:
            return outs[0].view(q.shape)
        return outs[0].view(q.shape), outs[1].view(k.shape)

    @staticmethod
    @once_differentiable
    def backward(ctx, *cotangents):
        *tensors, positions = ctx.saved_tensors
        # hooks on saved tensors may hand back other types and layouts
        q, k, *weights = (None if t is None else t.to(kind) for t, kind in zip(tensors, ctx.types))
        weights = [None if w is None else w.contiguous() for w in weights]
        cotangents = [*cotangents, None][:2]
        # a tensor without a cotangent has no gradient, nor has its weight
        rows = [None if g is None else _rows(t) for t, g in zip((q, k), cotangents)]
        cots = [None if g is None else _rows(g.to(q.dtype)) for g in cotangents]
        if cots[0] is None and cots[1] is None:
            return (None,) * 6
        if positions.dtype not in _POSITIONS:
            positions = positions.float()
        grads = list(_backward(rows[0], cots[0], rows[1], cots[1], *weights, positions, ctx.plan, ctx.needs_input_grad[:4]))
        for i, t in enumerate((q, k)):
            if cots[i] is None:
                grads[2 + i] = None
            elif grads[i] is not None:
                grads[i] = grads[i].view(t.shape)
        return (*grads, None, None)


def norm_rotary_embed(q, k, q_weight, k_weight, positions, sections, base=10000.0, shared_frequencies=False, interleaved=False, eps=1e-6):
    """Norms every head of ``q`` and ``k`` and rotates it by its token's positions: ``(q', k')``, or ``q'`` when ``k`` is None.

    A head's row ``x`` becomes ``x / sqrt(mean(x ** 2) + eps) * weight``, over all ``D`` channels, and is then rotated.

    Args:
        q: ``[..., H, D]`` float32 or bfloat16, ``D`` even, at most 256; strides are free.
        k: ``[..., Hk, D]`` with the same leading shape and type, or None.
        q_weight, k_weight: ``[D]`` float32 or bfloat16, both of one type, for all heads of ``q``, of ``k``; None: ones.
        positions, sections, base, shared_frequencies, interleaved: as in :func:`~rfdetr_jax_amd.rotary_embed`.
        eps: from ``2 ** -126`` to ``2 ** 126``.

    Differentiable in ``q``, ``k`` and the weights, not in ``positions``, which get no gradient. Sums are float32 (the
    weights' gradients over all tokens and heads too, in a fixed order), and every result is rounded once.

    Raises:
        ValueError: shapes, devices or sizes that do not fit.
        TypeError: types other than the above.
        RuntimeError: tensors that are not on a GPU.
    """
    sections = tuple(int(s) for s in sections)
    out = _native.binding().norm_rotary(q, k, q_weight, k_weight, positions, sections, base, bool(shared_frequencies), bool(interleaved), eps)
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
    if k is None and k_weight is not None:
        raise ValueError("k_weight without k")
    for name, w in (("q_weight", q_weight), ("k_weight", k_weight)):
        if w is None:
            continue
        if w.dtype not in _DTYPES:
            raise TypeError(f"{name} dtype {w.dtype} is not supported (float32 or bfloat16)")
        if tuple(w.shape) != (q.shape[-1],):
            raise ValueError(f"{name} must be [{q.shape[-1]}], got {tuple(w.shape)}")
        if w.device != q.device:
            raise ValueError(f"{name} is on {w.device}, the queries on {q.device}")
    if q_weight is not None and k_weight is not None and q_weight.dtype != k_weight.dtype:
        raise TypeError(f"the weights must be of one type, got {q_weight.dtype} and {k_weight.dtype}")
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
    base, eps = float(base), float(eps)
    if not 0.0 < base < float("inf"):
        raise ValueError(f"base must be positive and finite, got {base}")
    if not 2.0 ** -126 <= eps <= 2.0 ** 126:
        raise ValueError(f"eps must lie from 2^-126 to 2^126, got {eps}")
    return _NormRotary.apply(q, k, q_weight, k_weight, positions.flatten(0, -2) if positions.dim() > 1 else positions[None],
                             (sections, base, bool(shared_frequencies), bool(interleaved), eps))
