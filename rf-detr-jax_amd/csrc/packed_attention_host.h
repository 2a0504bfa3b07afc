// packed_attention_host.h — argument checks and parameters that the C entries of the packed attention and of the
// attention over a cache in 4 bits share.
#pragma once

#include "msda.h"
#include "packed_attention_launch.h"

namespace msda_host {

inline int64_t pk_slots(int64_t rows, int sequences) { return rows / msda::kPkTile + sequences + 2; }

inline int pk_shape(const msda::PackShape& s) {
  if (s.dtype != MSDA_DTYPE_F32 && s.dtype != MSDA_DTYPE_BF16) return fail(MSDA_ERR_UNSUPPORTED, "packed attention: unsupported dtype code %d", s.dtype);
  if (s.sequences < 0 || s.q_rows < 0 || s.k_rows < 0 || s.heads < 0 || s.kv_heads < 0)
    return fail(MSDA_ERR_INVALID_ARGUMENT, "packed attention: negative extent");
  if (s.head_dim < 8 || s.head_dim > 128 || s.head_dim % 8 != 0)
    return fail(MSDA_ERR_UNSUPPORTED, "packed attention: head_dim %d (multiples of 8 up to 128 supported)", s.head_dim);
  if (s.heads == 0 || s.kv_heads == 0 || s.heads % s.kv_heads != 0)
    return fail(MSDA_ERR_INVALID_ARGUMENT, "packed attention: %d heads do not divide into %d key heads", s.heads, s.kv_heads);
  if (s.heads / s.kv_heads > msda::kPkChunk)
    return fail(MSDA_ERR_UNSUPPORTED, "packed attention: %d query heads to a key head (at most %d)", s.heads / s.kv_heads, msda::kPkChunk);
  // row numbers of a key head's matrix, tiles included, are formed in 32 bits
  const int64_t group = s.heads / s.kv_heads, tiles = (static_cast<int64_t>(s.sequences) + 3) * msda::kPkTile;
  if (s.q_rows * group + tiles >= (int64_t{1} << 31) || s.k_rows + tiles >= (int64_t{1} << 31))
    return fail(MSDA_ERR_UNSUPPORTED, "packed attention: too many rows");
  return MSDA_OK;
}

// The window of the scores; the largest int where there is none.
inline int pk_window(const msda_score_shape* shape) { return shape == nullptr || shape->window == 0 ? 0x7fffffff : shape->window; }

template <int ntensors>
int pk_strides(const msda::PackShape& s, const int64_t* strides, const void* const (&tensors)[ntensors]) {
  if (strides == nullptr) return fail(MSDA_ERR_INVALID_ARGUMENT, "packed attention: NULL strides");
  const int64_t e = s.dtype == MSDA_DTYPE_BF16 ? 8 : 4;
  for (int i = 0; i < 2 * ntensors; ++i)
    if (strides[i] < 0 || strides[i] % e != 0)
      return fail(MSDA_ERR_INVALID_ARGUMENT, "packed attention: stride %d (%lld) must be a non-negative multiple of 16 bytes", i,
                  static_cast<long long>(strides[i]));
  // A tile's byte offsets are formed in 31 bits, its end from its rows: 64 rows, in the backward those of a group's heads
  const int64_t group = s.heads / s.kv_heads;
  for (int i = 0; i < ntensors; ++i)
    if (tensors[i] != nullptr || strides[2 * i] != 0 || strides[2 * i + 1] != 0)
      if (strides[2 * i] < s.head_dim || strides[2 * i] >= (int64_t{1} << 22) || ((i == 0 || i == 4) && strides[2 * i + 1] >= (int64_t{1} << 27) / group))
        return fail(MSDA_ERR_UNSUPPORTED, "packed attention: strides %lld, %lld of tensor %d: rows must lie head_dim to 2^22 elements apart, the heads of a group within 2^27",
                    static_cast<long long>(strides[2 * i]), static_cast<long long>(strides[2 * i + 1]), i);
  return MSDA_OK;
}

inline msda::PackParams pk_params(const msda::PackShape& s, const int32_t* q_offsets, const int32_t* k_offsets, const int32_t* k_lengths, const int64_t* strides,
                           int ntensors, const int* order, int causal, float scale) {
  msda::PackParams p{};
  p.q_offsets = q_offsets;
  p.k_offsets = k_offsets;
  p.k_lengths = k_lengths;
  p.sequences = s.sequences;
  p.q_rows = s.q_rows;
  p.k_rows = s.k_rows;
  p.heads = s.heads;
  p.kv_heads = s.kv_heads;
  p.group = s.heads / s.kv_heads;
  p.dim = s.head_dim;
  p.causal = causal != 0;
  p.splits = 1;
  p.scale = scale;
  p.scale2 = static_cast<float>(1.4426950408889634 * static_cast<double>(scale));
  for (int t = 0; t < ntensors; ++t)
    for (int j = 0; j < 2; ++j) p.st[order[t]][j] = strides[2 * t + j];
  return p;
}

inline int pk_scale(float scale) {
  // (the backward divides by it)
  if (!(scale >= 0x1p-64f && scale <= 0x1p64f)) return fail(MSDA_ERR_INVALID_ARGUMENT, "packed attention: scale %g must lie from 2^-64 to 2^64", static_cast<double>(scale));
  return MSDA_OK;
}

inline int pk_offsets(const int32_t* q_offsets, const int32_t* k_offsets, const int32_t* k_lengths) {
  if (q_offsets == nullptr || k_offsets == nullptr) return fail(MSDA_ERR_INVALID_ARGUMENT, "packed attention: NULL offsets");
  if (!aligned_to(q_offsets, 4) || !aligned_to(k_offsets, 4) || !aligned_to(k_lengths, 4))
    return fail(MSDA_ERR_INVALID_ARGUMENT, "packed attention: offsets and lengths must be aligned to 4 bytes");
  return MSDA_OK;
}

inline int pk_check_shape(const msda_score_shape* shape, int causal) {
  if (shape == nullptr) return MSDA_OK;
  if (shape->cap != 0.0f && !(shape->cap >= 0x1p-32f && shape->cap <= 0x1p32f))
    return fail(MSDA_ERR_INVALID_ARGUMENT, "packed attention: cap %g must be 0 or lie from 2^-32 to 2^32", static_cast<double>(shape->cap));
  if (shape->window < 0) return fail(MSDA_ERR_INVALID_ARGUMENT, "packed attention: window %d", shape->window);
  if (shape->prefix_lengths != nullptr && !causal) return fail(MSDA_ERR_INVALID_ARGUMENT, "packed attention: prefix lengths without causal");
  if (!aligned_to(shape->slopes, 4) || !aligned_to(shape->prefix_lengths, 4))
    return fail(MSDA_ERR_INVALID_ARGUMENT, "packed attention: slopes and prefix lengths must be aligned to 4 bytes");
  return MSDA_OK;
}

// Fills in the shape; the kernels that it needs (enum PackShaped), 0 for the plain ones.
inline int pk_set_shape(msda::PackParams& p, const msda_score_shape* shape) {
  p.window = pk_window(shape);
  if (shape == nullptr) return 0;
  int mod = shape->window != 0 || shape->prefix_lengths != nullptr ? msda::kPkRanges : 0;
  p.prefix = shape->prefix_lengths;
  if (shape->slopes != nullptr) {
    mod |= msda::kPkRanges | msda::kPkSlope;
    p.slopes = shape->slopes;
  }
  if (shape->cap != 0.0f) {
    mod |= msda::kPkRanges | msda::kPkCap;
    const double cap = shape->cap, inner = static_cast<double>(p.scale) / cap;
    p.inner = static_cast<float>(inner);
    p.cap2 = static_cast<float>(1.4426950408889634 * cap);
    p.bend = static_cast<float>(2.0 * 1.4426950408889634 * inner);
  }
  return mod;
}

}  // namespace msda_host
