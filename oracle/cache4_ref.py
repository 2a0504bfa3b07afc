"""CPU oracle for the cache in 4 bits — TEST INFRASTRUCTURE ONLY.

Nothing in the product path imports this module. NumPy, float64 from the given inputs, exact:

* ``encode``: rows ``[..., D]`` to ``(codes [..., 16 B] uint8, scales [..., B] uint8)``, by trying the exponents one after
  the other and the eight magnitudes of each channel, the nearest first, then the even code.
* ``decode``: what such rows stand for.

Attention over it is shaped_attention_ref over the decoded rows, with its bounds.
"""

from __future__ import annotations

import numpy as np

__all__ = ["MAGNITUDES", "encode", "decode"]

MAGNITUDES = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
LOW, HIGH, BAD = -120, 125, 255


def _blocks(x):
    x = np.asarray(x, np.float64)
    pad = -x.shape[-1] % 32
    x = np.concatenate([x, np.zeros((*x.shape[:-1], pad))], -1)
    return x.reshape(*x.shape[:-1], -1, 32)


def encode(x):
    x = _blocks(x)
    shape = x.shape
    codes, scales = np.zeros(shape, np.uint8), np.zeros(shape[:-1], np.uint8)
    for at in np.ndindex(*shape[:-1]):
        block = x[at]
        if not np.isfinite(block).all():
            scales[at] = BAD
            continue
        most = np.abs(block).max()
        e = LOW
        if most > 0:
            e = max(LOW, min(HIGH, int(np.floor(np.log2(most))) - 4))
            while e < HIGH and most > 7 * 2.0 ** e:
                e += 1
        scales[at] = e + 127
        for i, v in enumerate(np.abs(block) / 2.0 ** e):
            away = [abs(v - m) for m in MAGNITUDES]
            best = min(range(8), key=lambda c: (away[c], c % 2))
            codes[at][i] = best + (8 if np.signbit(block[i]) else 0)
    codes = codes.reshape(*shape[:-2], -1)
    return codes[..., 0::2] | codes[..., 1::2] << 4, scales


def decode(codes, scales, d):
    codes = np.stack([codes & 15, codes >> 4], -1).reshape(*codes.shape[:-1], -1)
    value = np.array(MAGNITUDES)[codes & 7] * np.where(codes & 8, -1.0, 1.0)
    scale = np.where(scales > HIGH + 127, np.nan, 2.0 ** (scales.astype(np.float64) - 127))
    return (value.reshape(*value.shape[:-1], -1, 32) * scale[..., None]).reshape(value.shape)[..., :d]
