// rotary_abi.hip — C ABI of the rotary positions (include/msda.h): validation, the frequency table, launch.
// Validation runs before any HIP call.
#include "msda.h"
#include "msda_launch.h"
#include "rotary_kernels.h"

#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>

namespace {

using msda_host::aligned_to;
using msda_host::fail;

template <typename T, int VEC, bool NEIGHBOURS>
int rot_launch(const msda::RotaryParams& p, hipStream_t st) {
  const int64_t grid = (static_cast<int64_t>(p.tokens) + p.per - 1) / p.per;
  const int lds = p.per * p.pairs * static_cast<int>(sizeof(float2));
  hipLaunchKernelGGL((msda::rotary_kernel<T, VEC, NEIGHBOURS>), dim3(static_cast<unsigned>(grid)), dim3(256), lds, st, p);
  return msda_host::check_launch("rotary positions");
}

// 16-byte pieces where every row, the pairs' halves and what passes lie on their boundaries, elements otherwise
template <typename T>
int rot_typed(const msda::RotaryParams& p, bool neighbours, hipStream_t st) {
  constexpr int E = 16 / static_cast<int>(sizeof(T));
  bool whole = p.dim % E == 0 && (neighbours ? (2 * p.pairs) % E == 0 : p.pairs % E == 0);
  for (int i = 0; i < 2; ++i) {
    whole = whole && aligned_to(p.x[i], 16) && aligned_to(p.y[i], 16);
    for (int j = 0; j < 2; ++j) whole = whole && p.xs[i][j] % E == 0 && p.ys[i][j] % E == 0;
  }
  if (!whole) return neighbours ? rot_launch<T, 1, true>(p, st) : rot_launch<T, 1, false>(p, st);
  return neighbours ? rot_launch<T, E / 2, true>(p, st) : rot_launch<T, E, false>(p, st);
}

}  // namespace

extern "C" int msda_rotary(const void* q, void* q_out, const void* k, void* k_out, int dtype, const void* positions, int position_type, int tokens,
                           int heads, int kv_heads, int head_dim, const int64_t* strides, const int64_t* position_strides, const int32_t* sections,
                           int axes, double base, int shared_frequencies, int interleaved, int inverse, void* stream) {
  msda_host::clear_error();
  if (dtype != MSDA_DTYPE_F32 && dtype != MSDA_DTYPE_BF16) return fail(MSDA_ERR_UNSUPPORTED, "rotary: unsupported dtype code %d", dtype);
  if (position_type < MSDA_POSITION_I32 || position_type > MSDA_POSITION_F32)
    return fail(MSDA_ERR_UNSUPPORTED, "rotary: unsupported position type code %d", position_type);
  if (tokens < 0 || heads < 0 || kv_heads < 0) return fail(MSDA_ERR_INVALID_ARGUMENT, "rotary: negative extent");
  if (head_dim < 2 || head_dim % 2 != 0 || head_dim > 2 * msda::kRotMaxPairs)
    return fail(MSDA_ERR_UNSUPPORTED, "rotary: head_dim %d (even, at most %d)", head_dim, 2 * msda::kRotMaxPairs);
  if (static_cast<int64_t>(heads) + kv_heads > (1 << 16)) return fail(MSDA_ERR_UNSUPPORTED, "rotary: more than 65536 heads");
  if (axes < 1 || axes > msda::kRotMaxAxes) return fail(MSDA_ERR_UNSUPPORTED, "rotary: %d axes (1 to %d supported)", axes, msda::kRotMaxAxes);
  if (sections == nullptr || strides == nullptr || position_strides == nullptr) return fail(MSDA_ERR_INVALID_ARGUMENT, "rotary: NULL sections or strides");
  if (!(base > 0.0) || !std::isfinite(base)) return fail(MSDA_ERR_INVALID_ARGUMENT, "rotary: base %g must be positive and finite", base);
  int64_t pairs = 0;
  for (int a = 0; a < axes; ++a) {
    if (sections[a] < 1) return fail(MSDA_ERR_INVALID_ARGUMENT, "rotary: section %d has %d pairs", a, sections[a]);
    pairs += sections[a];
  }
  if (2 * pairs > head_dim)
    return fail(MSDA_ERR_INVALID_ARGUMENT, "rotary: %lld pairs do not fit head_dim %d", static_cast<long long>(pairs), head_dim);
  for (int i = 0; i < 8; ++i)
    if (strides[i] < 0) return fail(MSDA_ERR_INVALID_ARGUMENT, "rotary: negative stride");
  if (position_strides[0] < 0 || position_strides[1] < 0) return fail(MSDA_ERR_INVALID_ARGUMENT, "rotary: negative stride");
  if (tokens == 0 || heads + kv_heads == 0) return MSDA_OK;
  const size_t e = dtype == MSDA_DTYPE_BF16 ? 2 : 4, pe = position_type == MSDA_POSITION_I64 ? 8 : 4;
  if (positions == nullptr || (heads != 0 && (q == nullptr || q_out == nullptr)) || (kv_heads != 0 && (k == nullptr || k_out == nullptr)))
    return fail(MSDA_ERR_INVALID_ARGUMENT, "msda_rotary: NULL tensor pointer");
  if (!aligned_to(q, e) || !aligned_to(q_out, e) || !aligned_to(k, e) || !aligned_to(k_out, e) || !aligned_to(positions, pe))
    return fail(MSDA_ERR_INVALID_ARGUMENT, "rotary: tensors must be aligned to their elements");

  msda::RotaryParams p{};
  p.x[0] = heads != 0 ? q : nullptr;
  p.y[0] = heads != 0 ? q_out : nullptr;
  p.x[1] = kv_heads != 0 ? k : nullptr;
  p.y[1] = kv_heads != 0 ? k_out : nullptr;
  for (int i = 0; i < 2; ++i)
    for (int j = 0; j < 2; ++j) {
      const bool used = (i == 0 ? heads : kv_heads) != 0;
      p.xs[i][j] = used ? strides[4 * i + j] : 0;
      p.ys[i][j] = used ? strides[4 * i + 2 + j] : 0;
    }
  p.positions = positions;
  p.ps[0] = position_strides[0];
  p.ps[1] = position_strides[1];
  p.position_type = position_type;
  p.tokens = tokens;
  p.heads[0] = heads;
  p.heads[1] = kv_heads;
  p.dim = head_dim;
  p.pairs = static_cast<int>(pairs);
  p.sign = inverse ? -1.0f : 1.0f;
  const double log_base = std::log(base);
  for (int a = 0, i = 0; a < axes; ++a)
    for (int j = 0; j < sections[a]; ++j, ++i) {
      const double exponent = shared_frequencies ? static_cast<double>(i) / static_cast<double>(pairs) : static_cast<double>(j) / sections[a];
      p.turns[i] = std::exp(-exponent * log_base) * 0.15915494309189533577;  // 1 / (2 pi)
      p.axis[i] = static_cast<uint8_t>(a);
    }
  // Tokens of a workgroup: few enough for four workgroups a CU, and at most 8 (the angles of 8 tokens keep
  // 256 threads busy for one or two steps).
  p.per = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(8, tokens / 1024)));
  hipStream_t st = static_cast<hipStream_t>(stream);
  return dtype == MSDA_DTYPE_BF16 ? rot_typed<msda::bf16_t>(p, interleaved != 0, st) : rot_typed<float>(p, interleaved != 0, st);
}
