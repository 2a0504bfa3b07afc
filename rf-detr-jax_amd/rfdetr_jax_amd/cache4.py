"""A cache of keys and values in 4 bits, and attention over it, on MI355X.

* :func:`new_cache4` — a :class:`Cache4` with room for some rows: 4.25 bits a channel, 68 bytes a row of 128 channels
  where bfloat16 takes 256.
* :func:`cache4_write` — the newest tokens' keys and values into it; :func:`cache4_read` — what rows of it stand for.
* :func:`cache4_attention` — :func:`~rfdetr_jax_amd.packed_attention` over it, for serving: one new token of each
  sequence, a chunk of a prompt, or both in one call.

All take the same offsets and lengths, which stay on the GPU: nothing is read back, and a step of writing and attending
can be captured into a graph and replayed with other lengths. HIP kernels (``msda_cache4_write`` / ``_read`` /
``_attention``); there is no CPU path and no gradient. No counterpart in the reference.

The numbers: 32 channels share a power of two, the least with every magnitude within 7 of it; a channel is the nearest of
0, 1/2, 1, 3/2, 2, 3, 4 and 6 times that, with its sign, the even code between two. A block that holds an infinity or NaN
reads as NaN.
"""

from __future__ import annotations

import ctypes
from typing import NamedTuple

import torch

from . import _native
from .packed_attention import _DTYPES, _Shape, _int32, _ptr, _rows16, _scale, _stream, _strides


class Cache4(NamedTuple):
    """Keys and values in 4 bits. With ``B = ceil(head_dim / 32)`` blocks of a row: ``keys`` and ``values`` uint8
    ``[Hk, rows, 16 B]``, two channels to a byte, the first in its lower half (sign 8, code 0 to 7); ``key_scales`` and
    ``value_scales`` uint8 ``[Hk, rows, B]``, the block's exponent + 127 (more than 252: not finite). All contiguous, on one GPU."""

    keys: torch.Tensor
    key_scales: torch.Tensor
    values: torch.Tensor
    value_scales: torch.Tensor
    head_dim: int

    @property
    def rows(self):
        return self.keys.shape[1]

    @property
    def kv_heads(self):
        return self.keys.shape[0]


def new_cache4(rows, kv_heads, head_dim, device):
    """A cache of zeros with room for ``rows`` rows (all sequences' room together)."""
    if head_dim % 8 or not 8 <= head_dim <= 128:
        raise ValueError(f"head_dim must be a multiple of 8 up to 128, got {head_dim}")
    if rows < 0 or kv_heads < 1:
        raise ValueError(f"a cache of {rows} rows and {kv_heads} heads")
    blocks = (head_dim + 31) // 32
    tensors = [torch.zeros((kv_heads, rows, n), dtype=torch.uint8, device=device) for n in (16 * blocks, blocks) * 2]
    return Cache4(*tensors, head_dim)


def _check_cache(cache):
    d = cache.head_dim
    if d % 8 or not 8 <= d <= 128:
        raise ValueError(f"head_dim must be a multiple of 8 up to 128, got {d}")
    if cache.keys.dim() != 3 or cache.kv_heads < 1:
        raise ValueError(f"the cache's keys must be [Hk, rows, bytes] with at least one head, got {tuple(cache.keys.shape)}")
    blocks = (d + 31) // 32
    for name, width in (("keys", 16 * blocks), ("key_scales", blocks), ("values", 16 * blocks), ("value_scales", blocks)):
        t = getattr(cache, name)
        if t.device.type != "cuda":
            raise RuntimeError(f"tensor on {t.device}; the HIP kernels need GPU tensors (there is no CPU path)")
        if t.dtype != torch.uint8:
            raise TypeError(f"the cache's {name} must be uint8, got {t.dtype}")
        if t.dim() != 3 or t.shape[2] != width or t.shape[:2] != cache.keys.shape[:2]:
            raise ValueError(f"the cache's {name} must be [Hk, rows, {width}], got {tuple(t.shape)}")
        if not t.is_contiguous() or t.data_ptr() % 16 and width != blocks:
            raise ValueError(f"the cache's {name} must be contiguous and aligned to 16 bytes")
        if t.device != cache.keys.device:
            raise ValueError(f"the cache's {name} are on {t.device}, its keys on {cache.keys.device}")
    if cache.rows >= 1 << 31:
        raise ValueError(f"the cache holds too many rows: {cache.rows}")


class _Places:
    def __init__(self, offsets, key_offsets, key_lengths, device):
        if offsets.dim() != 1 or offsets.numel() == 0:
            raise ValueError(f"offsets must be [sequences + 1], got {tuple(offsets.shape)}")
        self.count = offsets.numel() - 1
        self.q = _int32(offsets, (self.count + 1,), "offsets", device)
        self.k = self.q if key_offsets is None or key_offsets is offsets else _int32(key_offsets, (self.count + 1,), "key_offsets", device)
        self.lengths = None if key_lengths is None else _int32(key_lengths, (self.count,), "key_lengths", device)

    def pointers(self):
        return _ptr(self.q), _ptr(self.k), _ptr(self.lengths)


def _pointers(cache):
    return _ptr(cache.keys), _ptr(cache.key_scales), _ptr(cache.values), _ptr(cache.value_scales)


def _rows(cache, k, v, offsets, key_offsets, key_lengths, write):
    """Both ways of moving rows, on checked tensors."""
    places = _Places(offsets, key_offsets, key_lengths, cache.keys.device)
    ends = (*places.pointers(), places.count, k.shape[0], cache.rows, cache.kv_heads, cache.head_dim, _strides((k, v)), _stream(k.device))
    with torch.cuda.device(k.device):
        if write:
            rc = _native.lib().msda_cache4_write(_ptr(k), _ptr(v), _DTYPES[k.dtype], *_pointers(cache), *ends)
        else:
            rc = _native.lib().msda_cache4_read(*_pointers(cache), _ptr(k), _ptr(v), _DTYPES[k.dtype], *ends)
    _native.check(rc)


def cache4_write(cache, k, v, offsets, key_offsets=None, key_lengths=None):
    """Writes the keys and values of new tokens into ``cache``.

    Args:
        cache: a :class:`Cache4`.
        k, v: ``[T, Hk, D]`` float32 or bfloat16, the new tokens of all sequences behind one another.
        offsets: int32 ``[N + 1]`` on the same GPU: sequence ``i``'s new tokens are ``offsets[i]`` to
            ``offsets[i + 1] - 1`` (none, one or many).
        key_offsets: int32 ``[N + 1]``: its room in the cache, rows ``key_offsets[i]`` to ``key_offsets[i + 1] - 1``;
            ``offsets`` when None.
        key_lengths: int32 ``[N]``: how many rows of the room are keys, the new tokens included; all when None.

    The last new token becomes the last key. Tokens of no sequence, and those for which its keys leave no place, are
    skipped, and every other row stays as it is. Rooms must not overlap. No gradient flows through a cache.

    Raises:
        ValueError: shapes, devices or sizes that do not fit; tensors that need a gradient.
        TypeError: types other than the above.
        RuntimeError: tensors that are not on a GPU.
    """
    if _native.binding().cache4_rows(*cache, k, v, offsets, key_offsets, key_lengths, True) is not None:
        return
    _check_cache(cache)
    for name, t in (("k", k), ("v", v)):
        if t.device != cache.keys.device:
            raise ValueError(f"{name} is on {t.device}, the cache on {cache.keys.device}")
        if t.dtype not in _DTYPES:
            raise TypeError(f"{name} dtype {t.dtype} is not supported (float32 or bfloat16)")
        if t.dim() != 3 or tuple(t.shape[1:]) != (cache.kv_heads, cache.head_dim) or t.shape != k.shape:
            raise ValueError(f"k and v must be [T, {cache.kv_heads}, {cache.head_dim}], got {tuple(k.shape)} and {tuple(v.shape)}")
        if t.requires_grad and torch.is_grad_enabled():
            raise ValueError(f"{name} needs a gradient, which does not flow through a cache: pass it detached")
    if k.dtype != v.dtype:
        raise TypeError(f"k and v must be of one type, got {k.dtype} and {v.dtype}")
    _rows(cache, _rows16(k.detach()), _rows16(v.detach()), offsets, key_offsets, key_lengths, True)


def cache4_read(cache, tokens, offsets, key_offsets=None, key_lengths=None, dtype=torch.bfloat16):
    """``(k, v)``, ``[tokens, Hk, D]`` of ``dtype`` (float32 or bfloat16), what the newest rows of each sequence stand for,
    which both types hold exactly: the places of :func:`cache4_write`'s tokens, zeros for those without one.
    ``offsets`` that count all keys read whole sequences."""
    if dtype not in _DTYPES:
        raise TypeError(f"dtype {dtype} is not supported (float32 or bfloat16)")
    if not 0 <= tokens < 1 << 31:
        raise ValueError(f"{tokens} tokens")
    out = [torch.empty((tokens, cache.kv_heads, cache.head_dim), dtype=dtype, device=cache.keys.device) for _ in range(2)]
    if _native.binding().cache4_rows(*cache, *out, offsets, key_offsets, key_lengths, False) is not None:
        return tuple(out)
    _check_cache(cache)
    _rows(cache, *out, offsets, key_offsets, key_lengths, False)
    return tuple(out)


def cache4_attention(q, cache, offsets, key_offsets=None, key_lengths=None, causal=True, scale=None, *, cap=None, slopes=None, window=None,
                     prefix_lengths=None):
    """Softmax attention of packed queries over a cache in 4 bits: ``[T, H, D]`` in ``q``'s type.

    :func:`~rfdetr_jax_amd.packed_attention` with the values that ``cache`` holds for ``k`` and ``v``, and its arguments.
    ``q`` is float32 or bfloat16 ``[T, H, D]``, ``H`` a multiple of the cache's heads. The cache's values are bfloat16 numbers
    exactly and lose nothing more: results lie as far from the exact ones for these values as there.

    A batch whose sequences have up to 16 rows (tokens times ``H / Hk``) on average takes one kernel, others another. The first
    reads a sequence's keys once for each 16 of its rows, so a chunk among many single tokens is best called by itself: 63
    tokens and a chunk of 190 over 8,000 keys in bfloat16, 32 heads to 8, 639 us in one call, and with a chunk of 194, which
    the other kernel takes, 141.

    A query that sees no key, and rows outside every sequence, give zeros. Keys that are not seen take no part, whatever
    their rows hold; a block that is not finite makes the results of the queries that see it NaN (a key: all channels; a
    value: the block's). Not differentiable.

    Raises:
        ValueError: shapes, devices or sizes that do not fit; queries that need a gradient.
        TypeError: types other than the above.
        RuntimeError: tensors that are not on a GPU.
    """
    out = _native.binding().cache4_attention(q, *cache, offsets, key_offsets, key_lengths, bool(causal), scale, cap, slopes, window, prefix_lengths)
    if out is not None:
        return out
    _check_cache(cache)
    if q.device != cache.keys.device:
        raise ValueError(f"q is on {q.device}, the cache on {cache.keys.device}")
    if q.dtype not in _DTYPES:
        raise TypeError(f"attention dtype {q.dtype} is not supported (float32 or bfloat16)")
    if q.dim() != 3 or q.shape[2] != cache.head_dim:
        raise ValueError(f"q must be [rows, heads, {cache.head_dim}], got {tuple(q.shape)}")
    if max(q.shape) >= 1 << 31:
        raise ValueError(f"q is too large: {tuple(q.shape)}")
    if q.shape[1] == 0 or q.shape[1] % cache.kv_heads:
        raise ValueError(f"{q.shape[1]} query heads do not divide into {cache.kv_heads} key heads")
    if q.shape[1] > 64 * cache.kv_heads:
        raise ValueError(f"at most 64 query heads may share a key head, got {q.shape[1]} and {cache.kv_heads}")
    if q.requires_grad and torch.is_grad_enabled():
        raise ValueError("q needs a gradient, which attention over a cache in 4 bits does not give: pass it detached")
    places = _Places(offsets, key_offsets, key_lengths, q.device)
    shape = _Shape(cap, slopes, window, prefix_lengths, causal, q.shape[1], places.count, q.device)
    scale = _scale(scale, q.shape[2])
    q = _rows16(q.detach(), 64)
    out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    lib, code = _native.lib(), _DTYPES[q.dtype]
    dims = (places.count, q.shape[0], cache.rows, q.shape[1], cache.kv_heads, q.shape[2])
    with torch.cuda.device(q.device):
        nbytes = lib.msda_cache4_attention_workspace_size(code, *dims, shape.window)
        _native.check(min(nbytes, 0))
        ws = _native.workspace(nbytes, q.device) if nbytes else None
        rc = lib.msda_cache4_attention(_ptr(q), code, _ptr(out), *_pointers(cache), *places.pointers(), *dims, _strides((q, out)), int(causal), scale,
                                       shape.pointer(), _ptr(ws), nbytes, _stream(q.device))
    _native.check(rc)
    return out
