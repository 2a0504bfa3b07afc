// cache4_launch.h — host-side dispatch of the attention over a cache in 4 bits, shared by the translation units that
// instantiate its kernels (one per type and scores) and by the C ABI (cache4_abi.hip).
#pragma once

#include "cache4_kernels.h"
#include "packed_attention_launch.h"

namespace msda_host {

// Few rows a sequence (few), or tiles of 128; p.splits > 1: the join behind.
template <typename T, int DT, int MOD>
int c4_fwd(const msda::PackParams& p, bool few, hipStream_t st) {
  int rc;
  if (few)
    rc = pk_launch(msda::cache4_attention_kernel<T, DT, MOD != 0>, static_cast<int64_t>(p.splits) * (p.sequences + 1) * p.kv_heads, p, st, "attention over a cache in 4 bits");
  else
    rc = pk_launch(msda::pk_fwd_kernel<T, DT, MOD, true>, static_cast<int64_t>(p.slots) * p.splits * p.kv_heads, p, st, "attention over a cache in 4 bits (tiles)");
  if (rc != MSDA_OK || p.splits == 1) return rc;
  constexpr int LPR = DT <= 64 ? 16 : 32;
  return pk_launch(msda::pk_join_kernel<T, LPR>, (static_cast<int64_t>(p.q_rows) * p.heads + 256 / LPR - 1) / (256 / LPR), p, st,
                   "attention over a cache in 4 bits (join)");
}

template <typename T, int MOD>
int dispatch_c4_fwd(const msda::PackParams& p, bool few, hipStream_t st) {
  if (p.dim <= 32) return c4_fwd<T, 32, MOD>(p, few, st);
  if (p.dim <= 64) return c4_fwd<T, 64, MOD>(p, few, st);
  if (p.dim <= 96) return c4_fwd<T, 96, MOD>(p, few, st);
  return c4_fwd<T, 128, MOD>(p, few, st);
}

// Instantiated in cache4_attention_*.hip.
#define MSDA_C4_FWD(T, MOD) template int dispatch_c4_fwd<T, MOD>(const msda::PackParams&, bool, hipStream_t)
#ifndef MSDA_C4_INSTANTIATE
extern MSDA_C4_FWD(float, 0);
extern MSDA_C4_FWD(float, 4);
extern MSDA_C4_FWD(float, 5);
extern MSDA_C4_FWD(float, 6);
extern MSDA_C4_FWD(float, 7);
extern MSDA_C4_FWD(msda::bf16_t, 0);
extern MSDA_C4_FWD(msda::bf16_t, 4);
extern MSDA_C4_FWD(msda::bf16_t, 5);
extern MSDA_C4_FWD(msda::bf16_t, 6);
extern MSDA_C4_FWD(msda::bf16_t, 7);
#endif

}  // namespace msda_host
