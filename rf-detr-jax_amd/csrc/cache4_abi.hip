// cache4_abi.hip — C ABI of the cache in 4 bits (include/msda.h): validation, launch planning, launches. Validation
// runs before any HIP call.
#include "msda.h"
#include "cache4_launch.h"
#include "packed_attention_host.h"

#include <hip/hip_runtime.h>

#include <algorithm>

namespace {

using msda::PackShape;
using msda::PackSplit;
using msda_host::aligned_to;
using msda_host::fail;

// Few rows to a sequence on average: the kernel that takes 16 rows at a time and gives every wave keys of its own. More:
// tiles of 128 rows. A sequence of more rows than 16 reads its keys once for each 16 there. 16 rows and 32 rows of every
// sequence, 4 key heads of 128 channels, us a call by 16 rows at a time (and in tiles): 16 sequences of 4,000 keys 23 and
// 56 (34), 64 of 2,400 keys 27 and 51 (75), one of 16,000 keys 20 and 55 (28). The choice is the batch's, by its average: a chunk among
// single tokens pays for it (63 tokens and a chunk of 190 over 8,000 keys, 32 heads to 8, bf16: 639 us; of 194, in tiles: 141).
bool c4_few(const PackShape& s) { return static_cast<int64_t>(s.q_rows) * (s.heads / s.kv_heads) <= static_cast<int64_t>(16) * s.sequences; }

// The parts of a sequence's keys in the kernel of few rows: chunks of one, and how many at most.
PackSplit c4_split(const PackShape& s, int window) {
  if (!c4_few(s)) return msda::pk_split(s, window);
  if (s.sequences == 0) return PackSplit{1, 1 << 30};
  const int64_t chunks = (std::min(s.k_rows / s.sequences, msda::pk_in_window(window)) + msda::kPkChunk - 1) / msda::kPkChunk;  // of an average sequence
  // Parts of 16 chunks, 4 to a wave, are worth their join and even out caches of different fill; longer ones where those
  // alone would be several rounds of workgroups.
  const int64_t cells = static_cast<int64_t>(s.sequences) * s.kv_heads;
  const int64_t part = std::max<int64_t>(16, chunks * cells / 8192);
  return PackSplit{static_cast<int>(std::clamp<int64_t>((chunks + part - 1) / part, 1, msda::kPkMostParts)), static_cast<int>(part)};
}

int64_t c4_workspace(const PackShape& s, int window) {
  const int64_t parts = c4_split(s, window).most, rows = static_cast<int64_t>(s.q_rows) * s.heads;
  return parts == 1 ? 0 : (parts * (s.head_dim + 2) + 1) * rows * 4;
}

int c4_shape(const PackShape& s) {
  const int rc = msda_host::pk_shape(s);
  if (rc != MSDA_OK) return rc;
  if (s.sequences >= 1 << 24 || s.kv_heads >= 1 << 16) return fail(MSDA_ERR_UNSUPPORTED, "cache in 4 bits: too many sequences or key heads");
  return MSDA_OK;
}

struct Cache {
  const uint8_t* codes[2];
  const uint8_t* scales[2];
};

int c4_cache(const Cache& c, bool needed) {
  for (int i = 0; i < 2; ++i) {
    if (needed && (c.codes[i] == nullptr || c.scales[i] == nullptr)) return fail(MSDA_ERR_INVALID_ARGUMENT, "cache in 4 bits: NULL tensor pointer");
    if (!aligned_to(c.codes[i], 16)) return fail(MSDA_ERR_INVALID_ARGUMENT, "cache in 4 bits: codes must be aligned to 16 bytes");
  }
  return MSDA_OK;
}

// The parameters of writing and reading, checked.
int c4_rows(msda::Cache4Params& p, const void* const (&tensors)[2], int dtype, const Cache& cache, const int32_t* q_offsets, const int32_t* k_offsets,
            const int32_t* k_lengths, int sequences, int tokens, int rows, int kv_heads, int head_dim, const int64_t* strides) {
  int rc;
  if ((rc = c4_shape(PackShape{dtype, sequences, tokens, rows, kv_heads, kv_heads, head_dim})) != MSDA_OK) return rc;
  if (strides == nullptr) return fail(MSDA_ERR_INVALID_ARGUMENT, "cache in 4 bits: NULL strides");
  const int64_t e = dtype == MSDA_DTYPE_BF16 ? 8 : 4;
  for (int i = 0; i < 4; ++i)
    if (strides[i] < 0 || strides[i] % e != 0)
      return fail(MSDA_ERR_INVALID_ARGUMENT, "cache in 4 bits: stride %d (%lld) must be a non-negative multiple of 16 bytes", i, static_cast<long long>(strides[i]));
  if (tokens == 0) return MSDA_OK;
  if ((rc = msda_host::pk_offsets(q_offsets, k_offsets, k_lengths)) != MSDA_OK || (rc = c4_cache(cache, rows != 0)) != MSDA_OK) return rc;
  for (int i = 0; i < 2; ++i) {
    if (tensors[i] == nullptr) return fail(MSDA_ERR_INVALID_ARGUMENT, "cache in 4 bits: NULL tensor pointer");
    if (!aligned_to(tensors[i], 16)) return fail(MSDA_ERR_INVALID_ARGUMENT, "cache in 4 bits: tensors must be aligned to 16 bytes");
    p.codes[i] = const_cast<uint8_t*>(cache.codes[i]);
    p.scales[i] = const_cast<uint8_t*>(cache.scales[i]);
    for (int j = 0; j < 2; ++j) p.st[i][j] = strides[2 * i + j];
  }
  p.q_offsets = q_offsets;
  p.k_offsets = k_offsets;
  p.k_lengths = k_lengths;
  p.sequences = sequences;
  p.tokens = tokens;
  p.rows = rows;
  p.kv_heads = kv_heads;
  p.dim = head_dim;
  p.blocks = (head_dim + 31) / 32;
  return MSDA_OK;
}

template <typename K>
int c4_launch(K kernel, const msda::Cache4Params& p, hipStream_t st, const char* what) {
  const int64_t waves = (2 * static_cast<int64_t>(p.kv_heads) * p.blocks * 4 + 63) / 64, grid = (waves * p.tokens + 3) / 4;
  if (grid >= int64_t{1} << 24) return fail(MSDA_ERR_UNSUPPORTED, "cache in 4 bits: too many workgroups");  // a launch's threads are counted in 32 bits
  hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(grid)), dim3(256), 0, st, p);
  return msda_host::check_launch(what);
}

template <typename T>
int c4_run(const msda::PackParams& p, int mod, bool few, hipStream_t st) {
  switch (mod) {
    case 0: return msda_host::dispatch_c4_fwd<T, 0>(p, few, st);
    case 4: return msda_host::dispatch_c4_fwd<T, 4>(p, few, st);
    case 5: return msda_host::dispatch_c4_fwd<T, 5>(p, few, st);
    case 6: return msda_host::dispatch_c4_fwd<T, 6>(p, few, st);
    default: return msda_host::dispatch_c4_fwd<T, 7>(p, few, st);
  }
}

}  // namespace

extern "C" {

int msda_cache4_write(const void* k, const void* v, int dtype, uint8_t* keys, uint8_t* key_scales, uint8_t* values, uint8_t* value_scales,
                      const int32_t* q_offsets, const int32_t* k_offsets, const int32_t* k_lengths, int sequences, int tokens, int rows, int kv_heads,
                      int head_dim, const int64_t* strides, void* stream) {
  msda_host::clear_error();
  msda::Cache4Params p{};
  const int rc = c4_rows(p, {k, v}, dtype, Cache{{keys, values}, {key_scales, value_scales}}, q_offsets, k_offsets, k_lengths, sequences, tokens, rows,
                         kv_heads, head_dim, strides);
  if (rc != MSDA_OK || tokens == 0 || rows == 0) return rc;
  p.x[0] = k;
  p.x[1] = v;
  hipStream_t st = static_cast<hipStream_t>(stream);
  return dtype == MSDA_DTYPE_BF16 ? c4_launch(msda::cache4_write_kernel<msda::bf16_t>, p, st, "writing a cache in 4 bits")
                                  : c4_launch(msda::cache4_write_kernel<float>, p, st, "writing a cache in 4 bits");
}

int msda_cache4_read(const uint8_t* keys, const uint8_t* key_scales, const uint8_t* values, const uint8_t* value_scales, void* k, void* v, int dtype,
                     const int32_t* q_offsets, const int32_t* k_offsets, const int32_t* k_lengths, int sequences, int tokens, int rows, int kv_heads,
                     int head_dim, const int64_t* strides, void* stream) {
  msda_host::clear_error();
  msda::Cache4Params p{};
  const int rc = c4_rows(p, {k, v}, dtype, Cache{{keys, values}, {key_scales, value_scales}}, q_offsets, k_offsets, k_lengths, sequences, tokens, rows,
                         kv_heads, head_dim, strides);
  if (rc != MSDA_OK || tokens == 0) return rc;
  p.y[0] = k;
  p.y[1] = v;
  hipStream_t st = static_cast<hipStream_t>(stream);
  return dtype == MSDA_DTYPE_BF16 ? c4_launch(msda::cache4_read_kernel<msda::bf16_t>, p, st, "reading a cache in 4 bits")
                                  : c4_launch(msda::cache4_read_kernel<float>, p, st, "reading a cache in 4 bits");
}

int64_t msda_cache4_attention_workspace_size(int dtype, int sequences, int q_rows, int k_rows, int heads, int kv_heads, int head_dim, int window) {
  msda_host::clear_error();
  const PackShape s{dtype, sequences, q_rows, k_rows, heads, kv_heads, head_dim};
  const msda_score_shape shape{0.0f, window, nullptr, nullptr};
  int rc;
  if ((rc = c4_shape(s)) != MSDA_OK || (rc = msda_host::pk_check_shape(&shape, 1)) != MSDA_OK) return rc;
  return c4_workspace(s, msda_host::pk_window(&shape));
}

int msda_cache4_attention(const void* q, int dtype, void* out, const uint8_t* keys, const uint8_t* key_scales, const uint8_t* values,
                          const uint8_t* value_scales, const int32_t* q_offsets, const int32_t* k_offsets, const int32_t* k_lengths, int sequences,
                          int q_rows, int k_rows, int heads, int kv_heads, int head_dim, const int64_t* strides, int causal, float scale,
                          const msda_score_shape* shape, void* workspace, int64_t workspace_bytes, void* stream) {
  msda_host::clear_error();
  const PackShape s{dtype, sequences, q_rows, k_rows, heads, kv_heads, head_dim};
  int rc;
  if ((rc = c4_shape(s)) != MSDA_OK || (rc = msda_host::pk_strides<2>(s, strides, {q, out})) != MSDA_OK || (rc = msda_host::pk_scale(scale)) != MSDA_OK ||
      (rc = msda_host::pk_check_shape(shape, causal)) != MSDA_OK)
    return rc;
  if (q_rows == 0) return MSDA_OK;
  if ((rc = msda_host::pk_offsets(q_offsets, k_offsets, k_lengths)) != MSDA_OK || (rc = c4_cache(Cache{{keys, values}, {key_scales, value_scales}}, k_rows != 0)) != MSDA_OK)
    return rc;
  if (q == nullptr || out == nullptr) return fail(MSDA_ERR_INVALID_ARGUMENT, "msda_cache4_attention: NULL tensor pointer");
  if (!aligned_to(q, 16) || !aligned_to(out, 16)) return fail(MSDA_ERR_INVALID_ARGUMENT, "cache in 4 bits: tensors must be aligned to 16 bytes");
  static const int order[2] = {msda::kPkQ, msda::kPkO};
  msda::PackParams p = msda_host::pk_params(s, q_offsets, k_offsets, k_lengths, strides, 2, order, causal, scale);
  p.q = q;
  p.out = out;
  p.k = keys;
  p.v = values;
  p.k_scales = key_scales;
  p.v_scales = value_scales;
  const int mod = msda_host::pk_set_shape(p, shape);
  const PackSplit split = c4_split(s, p.window);
  p.slots = static_cast<int>(msda_host::pk_slots(static_cast<int64_t>(q_rows) * p.group, sequences));
  p.splits = split.most;
  p.part = split.part;
  if (p.splits > 1) {
    const int64_t need = c4_workspace(s, p.window);
    if (workspace == nullptr || workspace_bytes < need || !aligned_to(workspace, 16))
      return fail(MSDA_ERR_INVALID_ARGUMENT, "msda_cache4_attention: the workspace must hold %lld bytes, aligned to 16", static_cast<long long>(need));
    p.part_o = static_cast<float*>(workspace);
    p.part_ml = p.part_o + static_cast<int64_t>(p.splits) * q_rows * heads * head_dim;
    p.part_n = reinterpret_cast<int32_t*>(p.part_ml + static_cast<int64_t>(p.splits) * q_rows * heads * 2);
  }
  hipStream_t st = static_cast<hipStream_t>(stream);
  return dtype == MSDA_DTYPE_BF16 ? c4_run<msda::bf16_t>(p, mod, c4_few(s), st) : c4_run<float>(p, mod, c4_few(s), st);
}

}  // extern "C"
