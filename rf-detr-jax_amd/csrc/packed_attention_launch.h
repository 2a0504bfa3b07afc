// packed_attention_launch.h — host-side dispatch of the packed-sequence attention kernels, shared by the
// translation units that instantiate them (one per type, so the build compiles them in parallel) and by
// the C ABI (packed_attention_abi.hip).
#pragma once

#include "msda_launch.h"
#include "packed_attention_kernels.h"

namespace msda_host {

template <typename K>
int pk_launch(K kernel, int64_t grid, const msda::PackParams& p, hipStream_t st, const char* what) {
  if (grid >= (int64_t{1} << 31)) return fail(MSDA_ERR_UNSUPPORTED, "packed attention: too many workgroups");
  if (grid == 0) return MSDA_OK;
  hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(grid)), dim3(64 * msda::kPkWaves), 0, st, p);
  return check_launch(what);
}

template <typename T, int DT>
int pk_fwd(const msda::PackParams& p, hipStream_t st) {
  const int rc = pk_launch(msda::pk_fwd_kernel<T, DT>, static_cast<int64_t>(p.slots) * p.splits * p.kv_heads, p, st, "packed attention forward");
  if (rc != MSDA_OK || p.splits == 1) return rc;
  constexpr int LPR = DT <= 64 ? 16 : 32;
  return pk_launch(msda::pk_join_kernel<T, LPR>, (static_cast<int64_t>(p.q_rows) * p.heads + 256 / LPR - 1) / (256 / LPR), p, st,
                   "packed attention forward (join)");
}

// q_slots, k_slots: tiles of the queries' and of the keys' side; p.splits: parts of a key tile
template <typename T, int DT>
int pk_bwd(msda::PackParams p, int q_slots, int k_slots, hipStream_t st) {
  p.slots = q_slots;
  int rc = pk_launch(msda::pk_bwd_q_kernel<T, DT>, static_cast<int64_t>(q_slots) * p.kv_heads, p, st, "packed attention backward (queries)");
  if (rc != MSDA_OK || (p.gk == nullptr && p.gv == nullptr)) return rc;
  p.slots = k_slots;
  rc = pk_launch(msda::pk_bwd_kv_kernel<T, DT>, static_cast<int64_t>(k_slots) * p.splits * p.kv_heads, p, st,
                 "packed attention backward (keys, values)");
  if (rc != MSDA_OK || p.splits == 1) return rc;
  return pk_launch(msda::pk_join_kv_kernel<T>, static_cast<int64_t>(k_slots) * msda::kPkJoin, p, st, "packed attention backward (join)");
}

template <typename T>
int dispatch_pk_fwd(const msda::PackParams& p, hipStream_t st) {
  if (p.dim <= 32) return pk_fwd<T, 32>(p, st);
  if (p.dim <= 64) return pk_fwd<T, 64>(p, st);
  if (p.dim <= 96) return pk_fwd<T, 96>(p, st);
  return pk_fwd<T, 128>(p, st);
}

template <typename T>
int dispatch_pk_bwd(const msda::PackParams& p, int q_slots, int k_slots, hipStream_t st) {
  if (p.dim <= 32) return pk_bwd<T, 32>(p, q_slots, k_slots, st);
  if (p.dim <= 64) return pk_bwd<T, 64>(p, q_slots, k_slots, st);
  if (p.dim <= 96) return pk_bwd<T, 96>(p, q_slots, k_slots, st);
  return pk_bwd<T, 128>(p, q_slots, k_slots, st);
}

// Instantiated in packed_attention_{fwd,bwd}_{f32,bf16}.hip.
extern template int dispatch_pk_fwd<float>(const msda::PackParams&, hipStream_t);
extern template int dispatch_pk_fwd<msda::bf16_t>(const msda::PackParams&, hipStream_t);
extern template int dispatch_pk_bwd<float>(const msda::PackParams&, int, int, hipStream_t);
extern template int dispatch_pk_bwd<msda::bf16_t>(const msda::PackParams&, int, int, hipStream_t);

}  // namespace msda_host
