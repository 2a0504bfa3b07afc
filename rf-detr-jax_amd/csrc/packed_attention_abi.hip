// packed_attention_abi.hip — C ABI of the attention over packed sequences (include/msda.h): validation,
// launch planning, kernel launches. Validation runs before any HIP call.
#include "msda.h"
#include "packed_attention_launch.h"

#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>

namespace {

using msda_host::aligned_to;
using msda_host::fail;

using msda::PackShape;
using msda::PackSplit;
using msda::pk_split;

int64_t slots_of(int64_t rows, int sequences) { return rows / msda::kPkTile + sequences + 2; }

int pk_shape(const PackShape& s) {
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

int pk_bwd_shape(const PackShape& s) {
  const int rc = pk_shape(s);
  if (rc != MSDA_OK) return rc;
  // The key side forms the byte offsets of a tile's row numbers in 31 bits: at most 64 / group tokens of `heads` times 16 bytes.
  if (s.kv_heads >= 1 << 21) return fail(MSDA_ERR_UNSUPPORTED, "packed attention backward: %d key heads (fewer than 2^21 supported)", s.kv_heads);
  return MSDA_OK;
}

// Bytes of the split forward's parts: f32 sums, (m, l) of every row and part, the rows' numbers of parts.
int64_t pk_fwd_workspace(const PackShape& s) {
  const int64_t parts = pk_split(s).most, rows = static_cast<int64_t>(s.q_rows) * s.heads;
  return parts == 1 ? 0 : (parts * (s.head_dim + 2) + 1) * rows * 4;
}

// The number of workgroups that may share a tile of keys in the backward: a causal sequence's first keys are
// seen by all its rows, so with few tiles the longest one sets the time. A part is kPkPart chunks (more where
// that makes more than kMost parts, or the tiles alone are several rounds of workgroups).
int pk_parts(const PackShape& s) {
  constexpr int64_t kWant = 2048, kMost = 8;
  if (s.sequences == 0 || s.k_rows == 0) return 1;
  const int64_t tiles = std::min<int64_t>(s.k_rows, s.k_rows / msda::kPkTile + s.sequences) * s.kv_heads;
  // The rows of one sequence, if it is 4 times the average: a longer one takes longer parts, and batches of short
  // sequences start no second kernel (4 us).
  const int64_t rows = std::min<int64_t>(s.q_rows, 4 * (static_cast<int64_t>(s.q_rows) / s.sequences + 1));
  const int64_t chunks = rows * (s.heads / s.kv_heads) / msda::kPkChunk;
  return static_cast<int>(std::max<int64_t>(1, std::min({kWant / tiles, (chunks + msda::kPkPart - 1) / msda::kPkPart, kMost})));
}

// Bytes of the parts' f32 sums of dk and dv.
int64_t pk_bwd_workspace(const PackShape& s) {
  const int parts = pk_parts(s);
  return parts == 1 ? 0 : static_cast<int64_t>(parts) * 2 * s.k_rows * s.kv_heads * s.head_dim * 4;
}

template <int ntensors>
int pk_strides(const PackShape& s, const int64_t* strides, const void* const (&tensors)[ntensors]) {
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

msda::PackParams pk_params(const PackShape& s, const int32_t* q_offsets, const int32_t* k_offsets, const int32_t* k_lengths, const int64_t* strides,
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

int pk_scale(float scale) {
  // (the backward divides by it)
  if (!(scale >= 0x1p-64f && scale <= 0x1p64f)) return fail(MSDA_ERR_INVALID_ARGUMENT, "packed attention: scale %g must lie from 2^-64 to 2^64", static_cast<double>(scale));
  return MSDA_OK;
}

int pk_offsets(const int32_t* q_offsets, const int32_t* k_offsets, const int32_t* k_lengths) {
  if (q_offsets == nullptr || k_offsets == nullptr) return fail(MSDA_ERR_INVALID_ARGUMENT, "packed attention: NULL offsets");
  if (!aligned_to(q_offsets, 4) || !aligned_to(k_offsets, 4) || !aligned_to(k_lengths, 4))
    return fail(MSDA_ERR_INVALID_ARGUMENT, "packed attention: offsets and lengths must be aligned to 4 bytes");
  return MSDA_OK;
}

}  // namespace

extern "C" {

int64_t msda_packed_attention_fwd_workspace_size(int dtype, int sequences, int q_rows, int k_rows, int heads, int kv_heads, int head_dim) {
  msda_host::clear_error();
  const PackShape s{dtype, sequences, q_rows, k_rows, heads, kv_heads, head_dim};
  const int rc = pk_shape(s);
  return rc != MSDA_OK ? rc : pk_fwd_workspace(s);
}

int64_t msda_packed_attention_bwd_workspace_size(int dtype, int sequences, int q_rows, int k_rows, int heads, int kv_heads, int head_dim) {
  msda_host::clear_error();
  const PackShape s{dtype, sequences, q_rows, k_rows, heads, kv_heads, head_dim};
  const int rc = pk_bwd_shape(s);
  return rc != MSDA_OK ? rc : pk_bwd_workspace(s);
}

int msda_packed_attention_fwd(const void* q, const void* k, const void* v, int dtype, void* out, void* out_rest, float* stats,
                              const int32_t* q_offsets, const int32_t* k_offsets, const int32_t* k_lengths, int sequences, int q_rows, int k_rows, int heads, int kv_heads,
                              int head_dim, const int64_t* strides, int causal, float scale, void* workspace, int64_t workspace_bytes,
                              void* stream) {
  msda_host::clear_error();
  const PackShape s{dtype, sequences, q_rows, k_rows, heads, kv_heads, head_dim};
  int rc;
  if ((rc = pk_shape(s)) != MSDA_OK || (rc = pk_strides<4>(s, strides, {q, k, v, out})) != MSDA_OK || (rc = pk_scale(scale)) != MSDA_OK) return rc;
  if (q_rows == 0) return MSDA_OK;
  if ((rc = pk_offsets(q_offsets, k_offsets, k_lengths)) != MSDA_OK) return rc;
  if (q == nullptr || out == nullptr || (k_rows != 0 && (k == nullptr || v == nullptr)))
    return fail(MSDA_ERR_INVALID_ARGUMENT, "msda_packed_attention_fwd: NULL tensor pointer");
  if (!aligned_to(q, 16) || !aligned_to(k, 16) || !aligned_to(v, 16) || !aligned_to(out, 16) || !aligned_to(out_rest, 16) || !aligned_to(stats, 16))
    return fail(MSDA_ERR_INVALID_ARGUMENT, "packed attention: tensors must be aligned to 16 bytes");
  static const int order[4] = {msda::kPkQ, msda::kPkK, msda::kPkV, msda::kPkO};
  msda::PackParams p = pk_params(s, q_offsets, k_offsets, k_lengths, strides, 4, order, causal, scale);
  p.q = q;
  p.k = k;
  p.v = v;
  p.out = out;
  p.rest = dtype == MSDA_DTYPE_BF16 ? out_rest : nullptr;
  p.stats = stats;
  p.slots = static_cast<int>(slots_of(static_cast<int64_t>(q_rows) * p.group, sequences));
  const PackSplit split = pk_split(s);
  p.splits = split.most;
  p.part = split.part;
  if (p.splits > 1) {
    const int64_t need = pk_fwd_workspace(s);
    if (workspace == nullptr || workspace_bytes < need || !aligned_to(workspace, 16))
      return fail(MSDA_ERR_INVALID_ARGUMENT, "msda_packed_attention_fwd: the workspace must hold %lld bytes, aligned to 16", static_cast<long long>(need));
    p.part_o = static_cast<float*>(workspace);
    p.part_ml = p.part_o + static_cast<int64_t>(p.splits) * q_rows * heads * head_dim;
    p.part_n = reinterpret_cast<int32_t*>(p.part_ml + static_cast<int64_t>(p.splits) * q_rows * heads * 2);
  }
  hipStream_t st = static_cast<hipStream_t>(stream);
  return dtype == MSDA_DTYPE_BF16 ? msda_host::dispatch_pk_fwd<msda::bf16_t>(p, st) : msda_host::dispatch_pk_fwd<float>(p, st);
}

int msda_packed_attention_bwd_const(const void* q, const void* k, const void* v, const void* out, const void* out_rest, const float* stats,
                                    float* row_numbers, const void* grad_out, int dtype, void* grad_q, void* grad_k, void* grad_v,
                                    const int32_t* q_offsets, const int32_t* k_offsets, const int32_t* k_lengths, int sequences, int q_rows, int k_rows,
                                    int heads, int kv_heads, int head_dim, const int64_t* strides, int causal, float scale, void* workspace,
                                    int64_t workspace_bytes, void* stream) {
  msda_host::clear_error();
  const PackShape s{dtype, sequences, q_rows, k_rows, heads, kv_heads, head_dim};
  int rc;
  if ((rc = pk_bwd_shape(s)) != MSDA_OK || (rc = pk_strides<8>(s, strides, {q, k, v, out, grad_out, grad_q, grad_k, grad_v})) != MSDA_OK ||
      (rc = pk_scale(scale)) != MSDA_OK)
    return rc;
  if ((grad_q == nullptr && grad_k == nullptr && grad_v == nullptr) || (q_rows == 0 && k_rows == 0)) return MSDA_OK;
  if ((rc = pk_offsets(q_offsets, k_offsets, k_lengths)) != MSDA_OK) return rc;
  if ((q_rows != 0 && (q == nullptr || out == nullptr || stats == nullptr || grad_out == nullptr)) || (k_rows != 0 && (k == nullptr || v == nullptr)) ||
      (q_rows != 0 && row_numbers == nullptr && (grad_k != nullptr || grad_v != nullptr)))
    return fail(MSDA_ERR_INVALID_ARGUMENT, "msda_packed_attention_bwd: NULL tensor pointer");
  if (!aligned_to(q, 16) || !aligned_to(k, 16) || !aligned_to(v, 16) || !aligned_to(out, 16) || !aligned_to(out_rest, 16) || !aligned_to(stats, 16) ||
      !aligned_to(row_numbers, 16) || !aligned_to(grad_out, 16) || !aligned_to(grad_q, 16) || !aligned_to(grad_k, 16) || !aligned_to(grad_v, 16))
    return fail(MSDA_ERR_INVALID_ARGUMENT, "packed attention: tensors must be aligned to 16 bytes");
  static const int order[8] = {msda::kPkQ, msda::kPkK, msda::kPkV, msda::kPkO, msda::kPkGO, msda::kPkGQ, msda::kPkGK, msda::kPkGV};
  msda::PackParams p = pk_params(s, q_offsets, k_offsets, k_lengths, strides, 8, order, causal, scale);
  p.q = q;
  p.k = k;
  p.v = v;
  p.o = out;
  p.rest = dtype == MSDA_DTYPE_BF16 ? const_cast<void*>(out_rest) : nullptr;
  p.go = grad_out;
  p.gq = grad_q;
  p.gk = grad_k;
  p.gv = grad_v;
  p.stats = const_cast<float*>(stats);  // (the backward reads it)
  p.numbers = grad_k != nullptr || grad_v != nullptr ? row_numbers : nullptr;
  if (grad_k != nullptr || grad_v != nullptr) p.splits = pk_parts(s);
  if (p.splits > 1) {
    const int64_t need = pk_bwd_workspace(s);
    if (workspace == nullptr || workspace_bytes < need || !aligned_to(workspace, 16))
      return fail(MSDA_ERR_INVALID_ARGUMENT, "msda_packed_attention_bwd: the workspace must hold %lld bytes, aligned to 16", static_cast<long long>(need));
    p.part_kv = static_cast<float*>(workspace);
  }
  const int q_slots = q_rows == 0 ? 0 : static_cast<int>(slots_of(static_cast<int64_t>(q_rows) * p.group, sequences));
  const int k_slots = k_rows == 0 ? 0 : static_cast<int>(slots_of(k_rows, sequences));
  hipStream_t st = static_cast<hipStream_t>(stream);
  return dtype == MSDA_DTYPE_BF16 ? msda_host::dispatch_pk_bwd<msda::bf16_t>(p, q_slots, k_slots, st)
                                  : msda_host::dispatch_pk_bwd<float>(p, q_slots, k_slots, st);
}

int msda_packed_attention_bwd(const void* q, const void* k, const void* v, const void* out, const void* out_rest, float* stats,
                              const void* grad_out, int dtype, void* grad_q, void* grad_k, void* grad_v, const int32_t* q_offsets, const int32_t* k_offsets,
                              const int32_t* k_lengths, int sequences, int q_rows, int k_rows, int heads, int kv_heads, int head_dim,
                              const int64_t* strides, int causal, float scale, void* workspace, int64_t workspace_bytes, void* stream) {
  return msda_packed_attention_bwd_const(q, k, v, out, out_rest, stats, stats, grad_out, dtype, grad_q, grad_k, grad_v, q_offsets, k_offsets, k_lengths,
                                         sequences, q_rows, k_rows, heads, kv_heads, head_dim, strides, causal, scale, workspace, workspace_bytes, stream);
}

}  // extern "C"
