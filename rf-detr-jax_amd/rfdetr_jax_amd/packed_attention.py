"""Softmax attention over packed sequences of different lengths, on MI355X.

* :func:`packed_attention` — queries ``[T, H, D]`` and keys and values ``[S, Hk, D]`` of many sequences
  behind one another, ``H`` a multiple of ``Hk`` (each key head serves ``H / Hk`` query heads), causal or
  not, differentiable in q, k and v. With ``key_lengths`` the keys are a cache with room for more rows than
  it holds, and the queries its newest tokens (one each, or a chunk of a prompt).
  Scores may be capped by a tanh, fall with the distance of query and key, and end at a window; a prefix of a causal
  sequence may be seen by all its queries.
* :func:`packed_attention_forward` / :func:`packed_attention_backward` — the two directions without
  autograd.

The lengths stay on the GPU: nothing is read back, so a call can be captured into a graph and replayed
with other lengths. Both directions run in HIP kernels (``msda_packed_attention_fwd`` / ``_bwd_const``, shaped scores
in ``msda_packed_attention_shaped_fwd`` / ``_bwd``). There is no CPU path. No counterpart in the reference.
"""

from __future__ import annotations

import ctypes

import torch
from torch.autograd.function import once_differentiable

from . import _native

_DTYPES = {torch.float32: _native.DTYPE_F32, torch.bfloat16: _native.DTYPE_BF16}


def _ptr(t):
    return None if t is None else ctypes.c_void_p(t.data_ptr())


def _stream(device):
    return ctypes.c_void_p(torch.cuda.current_stream(device).cuda_stream)


def _rows16(t, group=1):
    """``t`` as the kernels read it: channels contiguous, rows on 16-byte boundaries and apart, the heads of a group
    within 2^27 elements (a copy where they are not)."""
    step, (row, head, channel) = 16 // t.element_size(), t.stride()
    if channel != 1 or row % step or head % step or t.data_ptr() % 16 or not t.shape[2] <= row < 1 << 22 or (group > 1 and head * group >= 1 << 27):
        t = torch.empty(t.shape, dtype=t.dtype, device=t.device).copy_(t)
    return t


def _int32(t, shape, what, device):
    if t.dtype not in (torch.int32, torch.int64):
        raise TypeError(f"{what} must be int32 (or int64), got {t.dtype}")
    if tuple(t.shape) != shape:
        raise ValueError(f"{what} must be {list(shape)}, got {tuple(t.shape)}")
    if t.device != device:
        raise ValueError(f"{what} is on {t.device}, the queries on {device}")
    return t.to(torch.int32).contiguous()


def _check(q, k, v):
    for name, t in zip("qkv", (q, k, v)):
        if t.device.type != "cuda":
            raise RuntimeError(f"tensor on {t.device}; the HIP kernels need GPU tensors (there is no CPU path)")
        if t.dtype not in _DTYPES:
            raise TypeError(f"attention dtype {t.dtype} is not supported (float32 or bfloat16)")
        if t.dim() != 3:
            raise ValueError(f"{name} must be [rows, heads, D], got {tuple(t.shape)}")
        if max(t.shape) >= 1 << 31:
            raise ValueError(f"{name} is too large: {tuple(t.shape)}")
    if k.dtype != q.dtype or v.dtype != q.dtype:
        raise TypeError(f"q, k and v must be of one type, got {q.dtype}, {k.dtype}, {v.dtype}")
    if k.device != q.device or v.device != q.device:
        raise ValueError(f"q, k and v must be on one device, got {q.device}, {k.device}, {v.device}")
    if k.shape != v.shape or k.shape[2] != q.shape[2]:
        raise ValueError(f"q [T, H, D] and k, v [S, Hk, D] expected, got {tuple(q.shape)}, {tuple(k.shape)}, {tuple(v.shape)}")
    if q.shape[1] == 0 or k.shape[1] == 0 or q.shape[1] % k.shape[1]:
        raise ValueError(f"{q.shape[1]} query heads do not divide into {k.shape[1]} key heads")
    if q.shape[1] > 64 * k.shape[1]:
        raise ValueError(f"at most 64 query heads may share a key head, got {q.shape[1]} and {k.shape[1]}")
    if q.shape[2] % 8 or not 8 <= q.shape[2] <= 128:
        raise ValueError(f"head_dim must be a multiple of 8 up to 128, got {q.shape[2]}")


class _Sequences:
    """The offsets of one call as the kernels read them."""

    def __init__(self, q, k, offsets, key_offsets, key_lengths):
        if offsets.dim() != 1 or offsets.numel() == 0:
            raise ValueError(f"offsets must be [sequences + 1], got {tuple(offsets.shape)}")
        self.count = offsets.numel() - 1
        self.q = _int32(offsets, (self.count + 1,), "offsets", q.device)
        if key_offsets is None or key_offsets is offsets:
            self.k = self.q
        else:
            self.k = _int32(key_offsets, (self.count + 1,), "key_offsets", q.device)
        self.lengths = None if key_lengths is None else _int32(key_lengths, (self.count,), "key_lengths", q.device)


def _no_gradient(slopes):
    if slopes is not None and slopes.requires_grad and torch.is_grad_enabled():
        raise ValueError("slopes get no gradient: pass them detached")


def _scale(scale, head_dim):
    scale = head_dim ** -0.5 if scale is None else float(scale)
    if not 2.0 ** -64 <= scale <= 2.0 ** 64:
        raise ValueError(f"scale must lie from 2^-64 to 2^64, got {scale}")
    return scale


class _Shape:
    """What the scores of one call are besides ``scale q.k``."""

    def __init__(self, cap, slopes, window, prefix_lengths, causal, heads, sequences, device):
        self.cap = 0.0 if cap is None else float(cap)
        if cap is not None and not 2.0 ** -32 <= self.cap <= 2.0 ** 32:
            raise ValueError(f"cap must lie from 2^-32 to 2^32, got {cap}")
        if window is not None and (int(window) != window or not 1 <= window < 1 << 31):
            raise ValueError(f"window must be a positive whole number, got {window}")
        self.window = 0 if window is None else int(window)
        if slopes is not None:
            if slopes.dtype != torch.float32:
                raise TypeError(f"slopes must be float32, got {slopes.dtype}")
            if tuple(slopes.shape) != (heads,):
                raise ValueError(f"slopes must be [{heads}], got {tuple(slopes.shape)}")
            if slopes.device != device:
                raise ValueError(f"slopes are on {slopes.device}, the queries on {device}")
            _no_gradient(slopes)
            slopes = slopes.detach().contiguous()
        self.slopes = slopes
        if prefix_lengths is not None:
            if not causal:
                raise ValueError("prefix_lengths belong to causal attention: without causal every query sees every key")
            prefix_lengths = _int32(prefix_lengths, (sequences,), "prefix_lengths", device)
        self.prefix = prefix_lengths
        self.any = self.cap != 0.0 or self.window != 0 or slopes is not None or prefix_lengths is not None

    def pointer(self):
        return ctypes.byref(_native.ScoreShape(self.cap, self.window, _ptr(self.slopes), _ptr(self.prefix)))


def _strides(tensors):
    flat = []
    for t in tensors:
        flat += [0, 0] if t is None else [t.stride(0), t.stride(1)]
    return (ctypes.c_int64 * len(flat))(*flat)


def _forward(q, k, v, seq, causal, scale, shape, backward):
    """``(out, rest, stats)``; with ``backward`` what it needs: what out's rounding left (bfloat16) and statistics."""
    out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    rest = torch.empty_like(out) if backward and q.dtype == torch.bfloat16 else None
    stats = torch.empty((q.shape[0], q.shape[1], 4), dtype=torch.float32, device=q.device) if backward else None
    lib, code = _native.lib(), _DTYPES[q.dtype]
    dims = (seq.count, q.shape[0], k.shape[0], q.shape[1], k.shape[1], q.shape[2])
    with torch.cuda.device(q.device):
        nbytes = lib.msda_packed_attention_shaped_fwd_workspace_size(code, *dims, shape.window)
        _native.check(min(nbytes, 0))
        ws = _native.workspace(nbytes, q.device) if nbytes else None
        rc = lib.msda_packed_attention_shaped_fwd(_ptr(q), _ptr(k), _ptr(v), code, _ptr(out), _ptr(rest), _ptr(stats), _ptr(seq.q), _ptr(seq.k),
                                                  _ptr(seq.lengths), *dims, _strides((q, k, v, out)), int(causal), scale, shape.pointer(),
                                                  _ptr(ws), nbytes, _stream(q.device))
    _native.check(rc)
    return out, rest, stats


def _backward(q, k, v, out, rest, stats, grad_out, seq, causal, scale, shape, needs):
    grads = [torch.empty(t.shape, dtype=t.dtype, device=t.device) if need else None for t, need in zip((q, k, v), needs)]
    lib, code = _native.lib(), _DTYPES[q.dtype]
    dims = (seq.count, q.shape[0], k.shape[0], q.shape[1], k.shape[1], q.shape[2])
    with torch.cuda.device(q.device):
        nbytes = 0
        if shape.any:
            nbytes = lib.msda_packed_attention_shaped_bwd_workspace_size(code, *dims, shape.window)
        elif needs[1] or needs[2]:
            nbytes = lib.msda_packed_attention_bwd_workspace_size(code, *dims)
        _native.check(min(nbytes, 0))
        ws = _native.workspace(nbytes, q.device) if nbytes else None
        numbers = torch.empty_like(stats) if needs[1] or needs[2] else None  # what the kernels hand on: other calls may read stats
        rc = lib.msda_packed_attention_shaped_bwd(_ptr(q), _ptr(k), _ptr(v), _ptr(out), _ptr(rest), _ptr(stats), _ptr(numbers), _ptr(grad_out), code,
                                                  *(_ptr(g) for g in grads), _ptr(seq.q), _ptr(seq.k), _ptr(seq.lengths), *dims,
                                                  _strides((q, k, v, out, grad_out, *grads)), int(causal), scale, shape.pointer(), _ptr(ws),
                                                  nbytes, _stream(q.device))
    _native.check(rc)
    return grads


def packed_attention_forward(q, k, v, offsets, key_offsets=None, key_lengths=None, causal=True, scale=None, *, cap=None, slopes=None,
                             window=None, prefix_lengths=None):
    """``(out, saved)`` of :func:`packed_attention`'s arguments, without autograd; ``saved`` is for
    :func:`packed_attention_backward`: the statistics ``[T, H, 4]``, and for bfloat16 what the rounding of ``out``
    left, ``[T, H, D]`` (else None)."""
    _check(q, k, v)
    seq = _Sequences(q, k, offsets, key_offsets, key_lengths)
    shape = _Shape(cap, slopes, window, prefix_lengths, causal, q.shape[1], seq.count, q.device)
    out, rest, stats = _forward(_rows16(q, 64), _rows16(k), _rows16(v), seq, causal, _scale(scale, q.shape[2]), shape, True)
    return out, (stats, rest)


def packed_attention_backward(q, k, v, out, saved, grad_out, offsets, key_offsets=None, key_lengths=None, causal=True, scale=None,
                              needs=(True, True, True), *, cap=None, slopes=None, window=None, prefix_lengths=None):
    """``(grad_q, grad_k, grad_v)``, contiguous, for the cotangent ``grad_out`` of ``out``; ``out`` and
    ``saved`` as :func:`packed_attention_forward` gave them, which are only read. None where ``needs`` says so."""
    _check(q, k, v)
    stats, rest = saved
    if any(t.shape != q.shape for t in (out, grad_out, *(() if rest is None else (rest,)))) or tuple(stats.shape) != (*q.shape[:2], 4):
        raise ValueError("out, its statistics or grad_out do not belong to these queries")
    if any(t.device != q.device for t in (out, grad_out, stats, *(() if rest is None else (rest,)))):
        raise ValueError("out, its statistics and grad_out must be on the queries' device")
    seq = _Sequences(q, k, offsets, key_offsets, key_lengths)
    shape = _Shape(cap, slopes, window, prefix_lengths, causal, q.shape[1], seq.count, q.device)
    # hooks on saved tensors may hand back other types and layouts: as the kernels read them
    q, k, v, out, grad_out = (_rows16(t.to(q.dtype), 64) for t in (q, k, v, out, grad_out))
    if rest is not None:
        out, rest = out.contiguous(), rest.to(q.dtype).contiguous()  # of the same strides
    stats = stats.to(torch.float32).contiguous()
    return tuple(_backward(q, k, v, out, rest, stats, grad_out, seq, causal, _scale(scale, q.shape[2]), shape, needs))


class _PackedAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, offsets, key_offsets, key_lengths, causal, scale, cap=None, slopes=None, window=None, prefix_lengths=None):
        _check(q, k, v)
        seq = _Sequences(q, k, offsets, key_offsets, key_lengths)
        shape = _Shape(cap, slopes, window, prefix_lengths, causal, q.shape[1], seq.count, q.device)
        scale = _scale(scale, q.shape[2])
        needs = any(ctx.needs_input_grad[:3])
        q, k, v = _rows16(q, 64), _rows16(k), _rows16(v)
        out, rest, stats = _forward(q, k, v, seq, causal, scale, shape, needs)
        if needs:
            ctx.save_for_backward(q, k, v, out, rest, stats, offsets, key_offsets, key_lengths, slopes, prefix_lengths)
            ctx.causal, ctx.scale, ctx.cap, ctx.window = causal, scale, cap, window
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_out):
        q, k, v, out, rest, stats, offsets, key_offsets, key_lengths, slopes, prefix_lengths = ctx.saved_tensors
        q, k, v = (t.to(grad_out.dtype) for t in (q, k, v))
        grads = packed_attention_backward(q, k, v, out, (stats, rest), grad_out, offsets, key_offsets, key_lengths, ctx.causal, ctx.scale,
                                          ctx.needs_input_grad[:3], cap=ctx.cap, slopes=None if slopes is None else slopes.float(), window=ctx.window,
                                          prefix_lengths=prefix_lengths)
        return (*grads, *[None] * 9)


def packed_attention(q, k, v, offsets, key_offsets=None, key_lengths=None, causal=True, scale=None, *, cap=None, slopes=None, window=None,
                     prefix_lengths=None):
    """Softmax attention of packed sequences: ``[T, H, D]`` in ``q``'s type (float32 or bfloat16).

    Args:
        q: ``[T, H, D]``, the queries of all sequences behind one another. ``D`` is a multiple of 8 up to 128.
        k, v: ``[S, Hk, D]``; query head ``h`` reads key head ``h // (H // Hk)``, which at most 64 share. All three
            may be views with larger row and head strides (slices of one projection).
        offsets: int32 ``[N + 1]`` on the same GPU: sequence ``i`` holds the queries ``offsets[i]`` to
            ``offsets[i + 1] - 1`` (none, one or many).
        key_offsets: the same for its keys; ``offsets`` when None.
        key_lengths: int32 ``[N]``: how many of the rows from ``key_offsets[i]`` on are keys (a cache with room
            for more); all of them when None.
        causal: query ``t`` of ``n`` sees the keys ``j <= t + m - n`` of ``m``, so that the last query sees every
            key; False: every key of its sequence.
        scale: of the scores, from ``2 ** -64`` to ``2 ** 64``; ``D ** -0.5`` when None.
        cap: a score ``s = scale q.k`` becomes ``cap tanh(s / cap)``; from ``2 ** -32`` to ``2 ** 32``.
        slopes: float32 ``[H]`` on the same GPU: behind the cap, head ``h``'s scores fall by ``slopes[h]`` for each place
            between query and key, ``|t + m - n - j|``. Finite; they get no gradient, and ones that need one are refused.
        window: keys at this distance and farther are not seen, on either side (1: a query's own place alone). What lies
            outside costs nothing.
        prefix_lengths: int32 ``[N]``, with ``causal``: the first so many keys of a sequence are seen by all its queries,
            the ones before them too (an image or a prompt before a text). A window bounds these, too.

    Documents that must not see each other are sequences of their own.

    Sums, softmax and statistics are float32. Of bfloat16 inputs the softmax weights and their gradients are rounded to
    bfloat16 for the matrix products: results lie 1.2 to 1.5 times as far from the exact ones as these rounded. Farther:
    gradients of k where a few tokens see a key, whose errors do not average out (4 to 31 tokens up to 1.8 times, two tokens
    2.4), and, without the options behind ``scale``, gradients of q and k of scores of several standard deviations (four: up
    to 1.9 times, of 8 channels 2.5). Where a row's gradients all but cancel (one weight near 1), what is left of them is good
    to 2^-16 of its terms. New tokens (a sequence's tokens times ``H / Hk`` up to 32) keep their weights in two
    bfloat16 numbers. Float32 inputs are float32 throughout. Calls whose work does not fill the GPU evenly take a workspace
    of partial sums, in float32 prompts up to some hundred MB (``msda_packed_attention_fwd_workspace_size``).

    A query that sees no key gives zeros. Rows of the result, and of the gradients, outside every sequence are
    zeros. Pairs that are not seen take no part, whatever their rows hold (infinities and NaN too; a key that is not
    finite makes the gradients of the queries that see it NaN, a query that is not, or its cotangent, those of the keys
    it sees). Offsets must rise and lie within the
    rows; they are not read back, and wrong ones give unspecified values.

    Raises:
        ValueError: shapes, devices or sizes that do not fit.
        TypeError: types other than the above.
        RuntimeError: tensors that are not on a GPU.
    """
    out = _native.binding().packed_attention(q, k, v, offsets, key_offsets, key_lengths, bool(causal), scale, cap, slopes, window, prefix_lengths)
    if out is not None:
        return out
    _no_gradient(slopes)  # here: inside an autograd function's forward no gradients are recorded
    return _PackedAttention.apply(q, k, v, offsets, key_offsets, key_lengths, bool(causal), scale, cap, slopes, window, prefix_lengths)
