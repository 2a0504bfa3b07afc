// packed_attention_abi.hip — C ABI of the attention over packed sequences (include/msda.h): validation,
// launch planning, kernel launches. Validation runs before any HIP call.
#include "msda.h"
#include "packed_attention_host.h"
#include "packed_attention_launch.h"

#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>

namespace {

using msda_host::aligned_to;
using msda_host::fail;
using msda_host::pk_check_shape;
using msda_host::pk_offsets;
using msda_host::pk_params;
using msda_host::pk_scale;
using msda_host::pk_set_shape;
using msda_host::pk_shape;
using msda_host::pk_slots;
using msda_host::pk_strides;
using msda_host::pk_window;

using msda::PackShape;
using msda::PackSplit;
using msda::pk_split;

int pk_bwd_shape(const PackShape& s) {
  const int rc = pk_shape(s);
  if (rc != MSDA_OK) return rc;
  // The key side forms the byte offsets of a tile's row numbers in 31 bits: at most 64 / group tokens of `heads` times 16 bytes.
  if (s.kv_heads >= 1 << 21) return fail(MSDA_ERR_UNSUPPORTED, "packed attention backward: %d key heads (fewer than 2^21 supported)", s.kv_heads);
  return MSDA_OK;
}

// Bytes of the split forward's parts: f32 sums, (m, l) of every row and part, the rows' numbers of parts.
int64_t pk_fwd_workspace(const PackShape& s, int window) {
  const int64_t parts = pk_split(s, window).most, rows = static_cast<int64_t>(s.q_rows) * s.heads;
  return parts == 1 ? 0 : (parts * (s.head_dim + 2) + 1) * rows * 4;
}

int pk_part(const PackShape& s, bool shaped) { return shaped && s.dtype == MSDA_DTYPE_F32 ? msda::kPkPartF32 : msda::kPkPart; }

// The number of workgroups that may share a tile of keys in the backward: a causal sequence's first keys are
// seen by all its rows, so with few tiles the longest one sets the time. A part is kPkPart chunks (more where
// that makes more than kMost parts, or the tiles alone are several rounds of workgroups).
int pk_parts(const PackShape& s, int window, bool shaped) {
  constexpr int64_t kWant = 2048, kMost = 8;
  if (s.sequences == 0 || s.k_rows == 0) return 1;
  const int64_t tiles = std::min<int64_t>(s.k_rows, s.k_rows / msda::kPkTile + s.sequences) * s.kv_heads;
  // Inside a window all tiles have about the same work: parts only where the tiles do not fill the CUs' two places
  // (12,093 tokens, 16 heads to 8 of 128 channels, a window of 1,024, 756 tiles: the join of two parts alone took 44 us).
  if (window < s.k_rows / s.sequences && tiles >= 512) return 1;
  // The rows of one sequence, if it is 4 times the average: a longer one takes longer parts, and batches of short
  // sequences start no second kernel (4 us).
  // No more than a window's see a tile.
  const int64_t rows = std::min<int64_t>({s.q_rows, 4 * (static_cast<int64_t>(s.q_rows) / s.sequences + 1), msda::pk_in_window(window)});
  const int64_t chunks = rows * (s.heads / s.kv_heads) / msda::kPkChunk, part = pk_part(s, shaped);
  return static_cast<int>(std::max<int64_t>(1, std::min({kWant / tiles, (chunks + part - 1) / part, kMost})));
}

// Workgroups that share a tile of queries in the backward of shaped scores: two to a CU where the tiles are fewer than
// the CUs, with 4 chunks of keys each at least (3,260 tokens of 8 heads, 32 channels, f32, 208 tiles: 86 us, in three parts 49 and 5 for their join).
int pk_q_parts(const PackShape& s, int window) {
  if (s.sequences == 0 || s.q_rows == 0) return 1;
  const int64_t rows = static_cast<int64_t>(s.q_rows) * (s.heads / s.kv_heads), tiles = std::min<int64_t>(rows, rows / msda::kPkTile + s.sequences) * s.kv_heads;
  const int64_t chunks = std::min(s.k_rows / s.sequences, msda::pk_in_window(window)) / msda::kPkChunk;
  return tiles >= 256 ? 1 : static_cast<int>(std::clamp<int64_t>(std::min((512 + tiles - 1) / tiles, chunks / 4), 1, 8));
}

// Bytes of the parts' f32 sums of dk and dv.
int64_t pk_kv_workspace(const PackShape& s, int window, bool shaped) {
  const int parts = pk_parts(s, window, shaped);
  return parts == 1 ? 0 : static_cast<int64_t>(parts) * 2 * s.k_rows * s.kv_heads * s.head_dim * 4;
}

// Those of dq, and the rows' numbers of parts.
int64_t pk_q_workspace(const PackShape& s, int window) {
  const int64_t parts = pk_q_parts(s, window);
  return parts == 1 ? 0 : (parts * s.head_dim + 1) * static_cast<int64_t>(s.q_rows) * s.heads * 4;
}

template <typename T>
int pk_run_fwd(const msda::PackParams& p, int mod, hipStream_t st) {
  switch (mod) {
    case 0: return msda_host::dispatch_pk_fwd<T, 0>(p, st);
    case 4: return msda_host::dispatch_pk_fwd<T, 4>(p, st);
    case 5: return msda_host::dispatch_pk_fwd<T, 5>(p, st);
    case 6: return msda_host::dispatch_pk_fwd<T, 6>(p, st);
    default: return msda_host::dispatch_pk_fwd<T, 7>(p, st);
  }
}

template <typename T>
int pk_run_bwd(const msda::PackParams& p, int mod, int q_slots, int k_slots, hipStream_t st) {
  switch (mod) {
    case 0: return msda_host::dispatch_pk_bwd<T, 0>(p, q_slots, k_slots, st);
    case 4: return msda_host::dispatch_pk_bwd<T, 4>(p, q_slots, k_slots, st);
    case 5: return msda_host::dispatch_pk_bwd<T, 5>(p, q_slots, k_slots, st);
    case 6: return msda_host::dispatch_pk_bwd<T, 6>(p, q_slots, k_slots, st);
    default: return msda_host::dispatch_pk_bwd<T, 7>(p, q_slots, k_slots, st);
  }
}

}  // namespace

extern "C" {

int64_t msda_packed_attention_fwd_workspace_size(int dtype, int sequences, int q_rows, int k_rows, int heads, int kv_heads, int head_dim) {
  msda_host::clear_error();
  const PackShape s{dtype, sequences, q_rows, k_rows, heads, kv_heads, head_dim};
  const int rc = pk_shape(s);
  return rc != MSDA_OK ? rc : pk_fwd_workspace(s, 0x7fffffff);
}

int64_t msda_packed_attention_bwd_workspace_size(int dtype, int sequences, int q_rows, int k_rows, int heads, int kv_heads, int head_dim) {
  msda_host::clear_error();
  const PackShape s{dtype, sequences, q_rows, k_rows, heads, kv_heads, head_dim};
  const int rc = pk_bwd_shape(s);
  return rc != MSDA_OK ? rc : pk_kv_workspace(s, 0x7fffffff, false);
}

int64_t msda_packed_attention_shaped_fwd_workspace_size(int dtype, int sequences, int q_rows, int k_rows, int heads, int kv_heads, int head_dim, int window) {
  msda_host::clear_error();
  const PackShape s{dtype, sequences, q_rows, k_rows, heads, kv_heads, head_dim};
  const msda_score_shape shape{0.0f, window, nullptr, nullptr};
  int rc;
  if ((rc = pk_shape(s)) != MSDA_OK || (rc = pk_check_shape(&shape, 1)) != MSDA_OK) return rc;
  return pk_fwd_workspace(s, pk_window(&shape));
}

int64_t msda_packed_attention_shaped_bwd_workspace_size(int dtype, int sequences, int q_rows, int k_rows, int heads, int kv_heads, int head_dim, int window) {
  msda_host::clear_error();
  const PackShape s{dtype, sequences, q_rows, k_rows, heads, kv_heads, head_dim};
  const msda_score_shape shape{0.0f, window, nullptr, nullptr};
  int rc;
  if ((rc = pk_bwd_shape(s)) != MSDA_OK || (rc = pk_check_shape(&shape, 1)) != MSDA_OK) return rc;
  // (of a call without a shape, too)
  return std::max(pk_kv_workspace(s, pk_window(&shape), true) + pk_q_workspace(s, pk_window(&shape)), pk_kv_workspace(s, pk_window(&shape), false));
}

int msda_packed_attention_shaped_fwd(const void* q, const void* k, const void* v, int dtype, void* out, void* out_rest, float* stats,
                                     const int32_t* q_offsets, const int32_t* k_offsets, const int32_t* k_lengths, int sequences, int q_rows, int k_rows, int heads, int kv_heads,
                                     int head_dim, const int64_t* strides, int causal, float scale, const msda_score_shape* shape,
                                            void* workspace, int64_t workspace_bytes, void* stream) {
  msda_host::clear_error();
  const PackShape s{dtype, sequences, q_rows, k_rows, heads, kv_heads, head_dim};
  int rc;
  if ((rc = pk_shape(s)) != MSDA_OK || (rc = pk_strides<4>(s, strides, {q, k, v, out})) != MSDA_OK || (rc = pk_scale(scale)) != MSDA_OK ||
      (rc = pk_check_shape(shape, causal)) != MSDA_OK)
    return rc;
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
  p.slots = static_cast<int>(pk_slots(static_cast<int64_t>(q_rows) * p.group, sequences));
  const int mod = pk_set_shape(p, shape);
  const PackSplit split = pk_split(s, p.window);
  p.splits = split.most;
  p.part = split.part;
  if (p.splits > 1) {
    const int64_t need = pk_fwd_workspace(s, p.window);
    if (workspace == nullptr || workspace_bytes < need || !aligned_to(workspace, 16))
      return fail(MSDA_ERR_INVALID_ARGUMENT, "msda_packed_attention_fwd: the workspace must hold %lld bytes, aligned to 16", static_cast<long long>(need));
    p.part_o = static_cast<float*>(workspace);
    p.part_ml = p.part_o + static_cast<int64_t>(p.splits) * q_rows * heads * head_dim;
    p.part_n = reinterpret_cast<int32_t*>(p.part_ml + static_cast<int64_t>(p.splits) * q_rows * heads * 2);
  }
  hipStream_t st = static_cast<hipStream_t>(stream);
  return dtype == MSDA_DTYPE_BF16 ? pk_run_fwd<msda::bf16_t>(p, mod, st) : pk_run_fwd<float>(p, mod, st);
}

int msda_packed_attention_fwd(const void* q, const void* k, const void* v, int dtype, void* out, void* out_rest, float* stats,
                              const int32_t* q_offsets, const int32_t* k_offsets, const int32_t* k_lengths, int sequences, int q_rows, int k_rows, int heads, int kv_heads,
                              int head_dim, const int64_t* strides, int causal, float scale, void* workspace, int64_t workspace_bytes,
                              void* stream) {
  return msda_packed_attention_shaped_fwd(q, k, v, dtype, out, out_rest, stats, q_offsets, k_offsets, k_lengths, sequences, q_rows, k_rows, heads, kv_heads,
                                          head_dim, strides, causal, scale, nullptr, workspace, workspace_bytes, stream);
}

int msda_packed_attention_shaped_bwd(const void* q, const void* k, const void* v, const void* out, const void* out_rest, const float* stats,
                                     float* row_numbers, const void* grad_out, int dtype, void* grad_q, void* grad_k, void* grad_v,
                                     const int32_t* q_offsets, const int32_t* k_offsets, const int32_t* k_lengths, int sequences, int q_rows, int k_rows,
                                     int heads, int kv_heads, int head_dim, const int64_t* strides, int causal, float scale, const msda_score_shape* shape,
                                     void* workspace, int64_t workspace_bytes, void* stream) {
  msda_host::clear_error();
  const PackShape s{dtype, sequences, q_rows, k_rows, heads, kv_heads, head_dim};
  int rc;
  if ((rc = pk_bwd_shape(s)) != MSDA_OK || (rc = pk_strides<8>(s, strides, {q, k, v, out, grad_out, grad_q, grad_k, grad_v})) != MSDA_OK ||
      (rc = pk_scale(scale)) != MSDA_OK || (rc = pk_check_shape(shape, causal)) != MSDA_OK)
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
  const int mod = pk_set_shape(p, shape);
  const bool keys = grad_k != nullptr || grad_v != nullptr;
  if (keys) p.splits = pk_parts(s, p.window, mod != 0);
  p.part = pk_part(s, mod != 0);
  p.q_parts = mod != 0 && grad_q != nullptr ? pk_q_parts(s, p.window) : 1;
  const int64_t kv_bytes = p.splits > 1 ? pk_kv_workspace(s, p.window, mod != 0) : 0, need = kv_bytes + (p.q_parts > 1 ? pk_q_workspace(s, p.window) : 0);
  if (need != 0) {
    if (workspace == nullptr || workspace_bytes < need || !aligned_to(workspace, 16))
      return fail(MSDA_ERR_INVALID_ARGUMENT, "msda_packed_attention_bwd: the workspace must hold %lld bytes, aligned to 16", static_cast<long long>(need));
    p.part_kv = static_cast<float*>(workspace);
    p.part_q = p.part_kv + kv_bytes / 4;
    p.part_q_n = reinterpret_cast<int32_t*>(p.part_q + static_cast<int64_t>(p.q_parts) * q_rows * heads * head_dim);
  }
  const int q_slots = q_rows == 0 ? 0 : static_cast<int>(pk_slots(static_cast<int64_t>(q_rows) * p.group, sequences));
  const int k_slots = k_rows == 0 ? 0 : static_cast<int>(pk_slots(k_rows, sequences));
  hipStream_t st = static_cast<hipStream_t>(stream);
  return dtype == MSDA_DTYPE_BF16 ? pk_run_bwd<msda::bf16_t>(p, mod, q_slots, k_slots, st) : pk_run_bwd<float>(p, mod, q_slots, k_slots, st);
}

int msda_packed_attention_bwd_const(const void* q, const void* k, const void* v, const void* out, const void* out_rest, const float* stats,
                                    float* row_numbers, const void* grad_out, int dtype, void* grad_q, void* grad_k, void* grad_v,
                                    const int32_t* q_offsets, const int32_t* k_offsets, const int32_t* k_lengths, int sequences, int q_rows, int k_rows,
                                    int heads, int kv_heads, int head_dim, const int64_t* strides, int causal, float scale, void* workspace,
                                    int64_t workspace_bytes, void* stream) {
  return msda_packed_attention_shaped_bwd(q, k, v, out, out_rest, stats, row_numbers, grad_out, dtype, grad_q, grad_k, grad_v, q_offsets, k_offsets, k_lengths,
                                          sequences, q_rows, k_rows, heads, kv_heads, head_dim, strides, causal, scale, nullptr, workspace, workspace_bytes, stream);
}

int msda_packed_attention_bwd(const void* q, const void* k, const void* v, const void* out, const void* out_rest, float* stats,
                              const void* grad_out, int dtype, void* grad_q, void* grad_k, void* grad_v, const int32_t* q_offsets, const int32_t* k_offsets,
                              const int32_t* k_lengths, int sequences, int q_rows, int k_rows, int heads, int kv_heads, int head_dim,
                              const int64_t* strides, int causal, float scale, void* workspace, int64_t workspace_bytes, void* stream) {
  return msda_packed_attention_bwd_const(q, k, v, out, out_rest, stats, stats, grad_out, dtype, grad_q, grad_k, grad_v, q_offsets, k_offsets, k_lengths,
                                         sequences, q_rows, k_rows, heads, kv_heads, head_dim, strides, causal, scale, workspace, workspace_bytes, stream);
}

}  // extern "C"
