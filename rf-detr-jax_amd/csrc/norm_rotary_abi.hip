// norm_rotary_abi.hip — C ABI of the norms with rotary positions (include/msda.h): validation, the frequency table,
// launch. Validation runs before any HIP call.
#include "msda.h"
#include "msda_launch.h"
#include "norm_rotary_kernels.h"

#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>

namespace {

using msda::NormRotaryParams;
using msda_host::aligned_to;
using msda_host::fail;

// Workgroups of the backward, each with one row of partial sums: four to a CU, as many as fit, where there are the tokens.
constexpr int64_t kMostGroups = 1024;

// Tokens of a step of a workgroup, which forms their angles together: few enough for four workgroups a CU and at most 8 in the
// forward (the angles of 8 tokens keep 256 threads busy for one or two steps), at most 16 in the backward, whose workgroups
// take several steps where that leaves tokens over: then smaller ones, so that all workgroups have about as many tokens (40
// heads of 128 channels, bf16, the weights' sums included: 16,384 tokens 123 us, 16,400 139 and 33,000 241; in steps of 16,
// a few workgroups with one more than the others, 171 and 274).
int tokens_of(int64_t tokens, bool backward) {
  if (!backward) return static_cast<int>(std::clamp<int64_t>(tokens / 1024, 1, 8));
  const int64_t steps = std::max<int64_t>(1, (tokens + 16 * kMostGroups - 1) / (16 * kMostGroups)), all = steps * kMostGroups;
  return static_cast<int>(std::max<int64_t>(1, (tokens + all - 1) / all));
}

int64_t groups_of(int64_t tokens, bool backward) {
  const int64_t per = tokens_of(tokens, backward), n = (tokens + per - 1) / per;
  return backward ? std::min(n, kMostGroups) : n;
}

template <typename T, int LPR, bool NEIGHBOURS>
void launch_pieces(const NormRotaryParams& p, bool backward, int64_t grid, int lds, hipStream_t st) {
  if (backward) hipLaunchKernelGGL((msda::norm_rotary_bwd_kernel<T, LPR, NEIGHBOURS>), dim3(static_cast<unsigned>(grid)), dim3(256), lds, st, p);
  else hipLaunchKernelGGL((msda::norm_rotary_kernel<T, LPR, NEIGHBOURS>), dim3(static_cast<unsigned>(grid)), dim3(256), lds, st, p);
}

// Lanes of 32 bytes where every row, the pairs' halves and what passes lie on 16-byte boundaries; elements otherwise.
template <typename T, bool NEIGHBOURS>
int run(const NormRotaryParams& p, bool backward, hipStream_t st) {
  constexpr int E = 16 / static_cast<int>(sizeof(T));
  bool whole = p.dim % E == 0 && (NEIGHBOURS ? 2 * p.pairs : p.pairs) % E == 0;
  for (int i = 0; i < 2; ++i) {
    whole = whole && aligned_to(p.x[i], 16) && aligned_to(p.y[i], 16) && aligned_to(p.dy[i], 16);
    for (int j = 0; j < 2; ++j) whole = whole && p.xs[i][j] % E == 0 && p.ys[i][j] % E == 0 && p.gs[i][j] % E == 0;
  }
  const int64_t grid = groups_of(p.tokens, backward);
  if (grid >= int64_t{1} << 24) return fail(MSDA_ERR_UNSUPPORTED, "norm rotary: too many tokens");  // a launch's threads are counted in 32 bits
  const int lds = p.per * p.pairs * static_cast<int>(sizeof(float2));
  if (!whole) {
    if (backward) hipLaunchKernelGGL((msda::norm_rotary_any_kernel<T, NEIGHBOURS, true>), dim3(static_cast<unsigned>(grid)), dim3(256), lds, st, p);
    else hipLaunchKernelGGL((msda::norm_rotary_any_kernel<T, NEIGHBOURS, false>), dim3(static_cast<unsigned>(grid)), dim3(256), lds, st, p);
  } else {
    const int turned = NEIGHBOURS ? 0 : p.pairs / E, units = turned + (p.dim - (NEIGHBOURS ? 0 : 2 * p.pairs) + 2 * E - 1) / (2 * E);
    if (units <= 4) launch_pieces<T, 4, NEIGHBOURS>(p, backward, grid, lds, st);
    else if (units <= 8) launch_pieces<T, 8, NEIGHBOURS>(p, backward, grid, lds, st);
    else if (units <= 16) launch_pieces<T, 16, NEIGHBOURS>(p, backward, grid, lds, st);
    else launch_pieces<T, 32, NEIGHBOURS>(p, backward, grid, lds, st);
  }
  return msda_host::check_launch(backward ? "norm and rotary positions (backward)" : "norm and rotary positions");
}

template <typename T>
int run(const NormRotaryParams& p, bool backward, bool neighbours, hipStream_t st) {
  return neighbours ? run<T, true>(p, backward, st) : run<T, false>(p, backward, st);
}

// The checks and parameters that both directions share; p.tokens 0: nothing to do.
int plan(NormRotaryParams& p, int dtype, const void* positions, int position_type, int weight_type, int tokens, int heads, int kv_heads, int head_dim,
         const int64_t* strides, int nstrides, const int64_t* position_strides, const int32_t* sections, int axes, double base, int shared_frequencies,
         double eps, bool backward) {
  if (dtype != MSDA_DTYPE_F32 && dtype != MSDA_DTYPE_BF16) return fail(MSDA_ERR_UNSUPPORTED, "norm rotary: unsupported dtype code %d", dtype);
  if (weight_type != MSDA_DTYPE_F32 && weight_type != MSDA_DTYPE_BF16) return fail(MSDA_ERR_UNSUPPORTED, "norm rotary: unsupported weight type code %d", weight_type);
  if (position_type < MSDA_POSITION_I32 || position_type > MSDA_POSITION_F32)
    return fail(MSDA_ERR_UNSUPPORTED, "norm rotary: unsupported position type code %d", position_type);
  if (tokens < 0 || heads < 0 || kv_heads < 0) return fail(MSDA_ERR_INVALID_ARGUMENT, "norm rotary: negative extent");
  if (head_dim < 2 || head_dim % 2 != 0 || head_dim > 2 * msda::kRotMaxPairs)
    return fail(MSDA_ERR_UNSUPPORTED, "norm rotary: head_dim %d (even, at most %d)", head_dim, 2 * msda::kRotMaxPairs);
  if (static_cast<int64_t>(heads) + kv_heads > (1 << 16)) return fail(MSDA_ERR_UNSUPPORTED, "norm rotary: more than 65536 heads");
  if (axes < 1 || axes > msda::kRotMaxAxes) return fail(MSDA_ERR_UNSUPPORTED, "norm rotary: %d axes (1 to %d supported)", axes, msda::kRotMaxAxes);
  if (sections == nullptr || strides == nullptr || position_strides == nullptr) return fail(MSDA_ERR_INVALID_ARGUMENT, "norm rotary: NULL sections or strides");
  if (!(base > 0.0) || !std::isfinite(base)) return fail(MSDA_ERR_INVALID_ARGUMENT, "norm rotary: base %g must be positive and finite", base);
  if (!(eps >= 0x1p-126 && eps <= 0x1p126)) return fail(MSDA_ERR_INVALID_ARGUMENT, "norm rotary: eps %g must lie from 2^-126 to 2^126", eps);
  int64_t pairs = 0;
  for (int a = 0; a < axes; ++a) {
    if (sections[a] < 1) return fail(MSDA_ERR_INVALID_ARGUMENT, "norm rotary: section %d has %d pairs", a, sections[a]);
    pairs += sections[a];
  }
  if (2 * pairs > head_dim)
    return fail(MSDA_ERR_INVALID_ARGUMENT, "norm rotary: %lld pairs do not fit head_dim %d", static_cast<long long>(pairs), head_dim);
  for (int i = 0; i < nstrides; ++i)
    if (strides[i] < 0) return fail(MSDA_ERR_INVALID_ARGUMENT, "norm rotary: negative stride");
  if (position_strides[0] < 0 || position_strides[1] < 0) return fail(MSDA_ERR_INVALID_ARGUMENT, "norm rotary: negative stride");
  p.positions = positions;
  p.ps[0] = position_strides[0];
  p.ps[1] = position_strides[1];
  p.position_type = position_type;
  p.weight_type = weight_type;
  p.tokens = heads + kv_heads == 0 ? 0 : tokens;
  p.heads[0] = heads;
  p.heads[1] = kv_heads;
  p.dim = head_dim;
  p.pairs = static_cast<int>(pairs);
  p.per = tokens_of(tokens, backward);
  p.eps = static_cast<float>(eps);
  p.inverse_dim = 1.0f / static_cast<float>(head_dim);
  const double log_base = std::log(base);
  for (int a = 0, i = 0; a < axes; ++a)
    for (int j = 0; j < sections[a]; ++j, ++i) {
      const double exponent = shared_frequencies ? static_cast<double>(i) / static_cast<double>(pairs) : static_cast<double>(j) / sections[a];
      p.turns[i] = std::exp(-exponent * log_base) * 0.15915494309189533577;  // 1 / (2 pi)
      p.axis[i] = static_cast<uint8_t>(a);
    }
  return MSDA_OK;
}

// Fills in a tensor that its heads use; its element size and strides as the kernels take them.
int put(const void* tensor, const int64_t* strides, size_t size, bool used, const void*& to, int64_t (&st)[2]) {
  to = used ? tensor : nullptr;
  for (int j = 0; j < 2; ++j) st[j] = to != nullptr ? strides[j] : 0;
  return aligned_to(to, size) ? MSDA_OK : fail(MSDA_ERR_INVALID_ARGUMENT, "norm rotary: tensors must be aligned to their elements");
}

}  // namespace

extern "C" {

int msda_norm_rotary_fwd(const void* q, void* q_out, const void* k, void* k_out, int dtype, const void* q_weight, const void* k_weight, int weight_type,
                         const void* positions, int position_type, int tokens, int heads, int kv_heads, int head_dim, const int64_t* strides,
                         const int64_t* position_strides, const int32_t* sections, int axes, double base, int shared_frequencies, int interleaved,
                         double eps, void* stream) {
  msda_host::clear_error();
  NormRotaryParams p{};
  int rc = plan(p, dtype, positions, position_type, weight_type, tokens, heads, kv_heads, head_dim, strides, 8, position_strides, sections, axes, base,
                shared_frequencies, eps, false);
  if (rc != MSDA_OK || p.tokens == 0) return rc;
  const size_t e = dtype == MSDA_DTYPE_BF16 ? 2 : 4, pe = position_type == MSDA_POSITION_I64 ? 8 : 4, we = weight_type == MSDA_DTYPE_BF16 ? 2 : 4;
  if (positions == nullptr || (heads != 0 && (q == nullptr || q_out == nullptr)) || (kv_heads != 0 && (k == nullptr || k_out == nullptr)))
    return fail(MSDA_ERR_INVALID_ARGUMENT, "msda_norm_rotary_fwd: NULL tensor pointer");
  if (!aligned_to(positions, pe) || !aligned_to(q_weight, we) || !aligned_to(k_weight, we))
    return fail(MSDA_ERR_INVALID_ARGUMENT, "norm rotary: tensors must be aligned to their elements");
  const void* out[2];
  if ((rc = put(q, strides, e, heads != 0, p.x[0], p.xs[0])) != MSDA_OK || (rc = put(q_out, strides + 2, e, heads != 0, out[0], p.ys[0])) != MSDA_OK ||
      (rc = put(k, strides + 4, e, kv_heads != 0, p.x[1], p.xs[1])) != MSDA_OK || (rc = put(k_out, strides + 6, e, kv_heads != 0, out[1], p.ys[1])) != MSDA_OK)
    return rc;
  for (int i = 0; i < 2; ++i) p.y[i] = const_cast<void*>(out[i]);
  p.w[0] = q_weight;
  p.w[1] = k_weight;
  hipStream_t st = static_cast<hipStream_t>(stream);
  return dtype == MSDA_DTYPE_BF16 ? run<msda::bf16_t>(p, false, interleaved != 0, st) : run<float>(p, false, interleaved != 0, st);
}

int64_t msda_norm_rotary_bwd_workspace_size(int tokens, int head_dim) {
  msda_host::clear_error();
  if (tokens < 0) return fail(MSDA_ERR_INVALID_ARGUMENT, "norm rotary: negative extent");
  if (head_dim < 2 || head_dim % 2 != 0 || head_dim > 2 * msda::kRotMaxPairs)
    return fail(MSDA_ERR_UNSUPPORTED, "norm rotary: head_dim %d (even, at most %d)", head_dim, 2 * msda::kRotMaxPairs);
  return groups_of(tokens, true) * 2 * head_dim * 4;
}

int msda_norm_rotary_bwd(const void* q, const void* grad_q_out, void* grad_q, const void* k, const void* grad_k_out, void* grad_k, int dtype,
                         const void* q_weight, const void* k_weight, void* grad_q_weight, void* grad_k_weight, int weight_type, const void* positions,
                         int position_type, int tokens, int heads, int kv_heads, int head_dim, const int64_t* strides, const int64_t* position_strides,
                         const int32_t* sections, int axes, double base, int shared_frequencies, int interleaved, double eps, void* workspace,
                         int64_t workspace_bytes, void* stream) {
  msda_host::clear_error();
  NormRotaryParams p{};
  int rc = plan(p, dtype, positions, position_type, weight_type, tokens, heads, kv_heads, head_dim, strides, 12, position_strides, sections, axes, base,
                shared_frequencies, eps, true);
  if (rc != MSDA_OK) return rc;
  const bool sums = grad_q_weight != nullptr || grad_k_weight != nullptr;
  const size_t e = dtype == MSDA_DTYPE_BF16 ? 2 : 4, pe = position_type == MSDA_POSITION_I64 ? 8 : 4, we = weight_type == MSDA_DTYPE_BF16 ? 2 : 4;
  if (!aligned_to(positions, pe) || !aligned_to(q_weight, we) || !aligned_to(k_weight, we) || !aligned_to(grad_q_weight, we) || !aligned_to(grad_k_weight, we))
    return fail(MSDA_ERR_INVALID_ARGUMENT, "norm rotary: tensors must be aligned to their elements");
  int64_t rows = 0;
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (p.tokens != 0) {
    if (positions == nullptr || (heads != 0 && (q == nullptr || grad_q_out == nullptr)) || (kv_heads != 0 && (k == nullptr || grad_k_out == nullptr)))
      return fail(MSDA_ERR_INVALID_ARGUMENT, "msda_norm_rotary_bwd: NULL tensor pointer");
    const void* out[2];
    if ((rc = put(q, strides, e, heads != 0, p.x[0], p.xs[0])) != MSDA_OK || (rc = put(grad_q_out, strides + 2, e, heads != 0, p.dy[0], p.gs[0])) != MSDA_OK ||
        (rc = put(grad_q, strides + 4, e, heads != 0, out[0], p.ys[0])) != MSDA_OK || (rc = put(k, strides + 6, e, kv_heads != 0, p.x[1], p.xs[1])) != MSDA_OK ||
        (rc = put(grad_k_out, strides + 8, e, kv_heads != 0, p.dy[1], p.gs[1])) != MSDA_OK || (rc = put(grad_k, strides + 10, e, kv_heads != 0, out[1], p.ys[1])) != MSDA_OK)
      return rc;
    for (int i = 0; i < 2; ++i) p.y[i] = const_cast<void*>(out[i]);
    p.w[0] = q_weight;
    p.w[1] = k_weight;
    rows = groups_of(tokens, true);
    if (sums) {
      const int64_t need = rows * 2 * head_dim * 4;
      if (workspace == nullptr || workspace_bytes < need || !aligned_to(workspace, 16))
        return fail(MSDA_ERR_INVALID_ARGUMENT, "msda_norm_rotary_bwd: the workspace must hold %lld bytes, aligned to 16", static_cast<long long>(need));
      p.part = static_cast<float*>(workspace);
    }
    rc = dtype == MSDA_DTYPE_BF16 ? run<msda::bf16_t>(p, true, interleaved != 0, st) : run<float>(p, true, interleaved != 0, st);
    if (rc != MSDA_OK) return rc;
  }
  if (!sums) return MSDA_OK;
  // (without tokens the sums are zeros)
  hipLaunchKernelGGL(msda::norm_rotary_join_kernel, dim3((2 * head_dim + 15) / 16), dim3(1024), 0, st, p.part, static_cast<int>(rows), head_dim, grad_q_weight,
                     grad_k_weight, weight_type);
  return msda_host::check_launch("norm and rotary positions (weights)");
}

}  // extern "C"
