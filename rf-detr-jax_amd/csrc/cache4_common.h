// cache4_common.h — the numbers of a cache of keys and values in 4 bits.
//
// The numbers. 32 channels of a row share a power of two 2^e, one byte e + 127; a channel is a sign and 3 bits for
// {0, 1/2, 1, 3/2, 2, 3, 4, 6} of it. e is the least with every magnitude within 7 2^e (6 and what rounds to it), from
// -120 to 125; a channel goes to the nearest, to the even code between two. A block that holds an infinity or NaN reads
// as NaN (byte 255; 253 and 254, which no block gets, do too). Every value is a bf16 number exactly, so that products on bf16 matrix instructions lose nothing.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

#include "attention_common.h"

namespace msda {

typedef __bf16 c4_bf2 __attribute__((ext_vector_type(2)));
typedef float c4_f2 __attribute__((ext_vector_type(2)));

// The scale of a block that is not finite as it is written, and the largest of one that is: what lies between (in memory that
// nothing wrote) would be values past bf16's largest, infinities, and counts as not finite.
constexpr uint32_t kC4Bad = 255, kC4Most = 252;

__device__ __forceinline__ float c4_scale(uint32_t byte) { return __uint_as_float(byte << 23); }

// 8 codes of one block as bf16.
__device__ __forceinline__ at_bf8 c4_bf16(uint32_t codes, float scale) {
  const c4_bf2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 0), b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 1);
  const c4_bf2 c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 2), d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 3);
  return at_bf8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}
__device__ __forceinline__ void c4_f32(uint32_t codes, float scale, float* v) {
  const c4_f2 a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes, scale, 0), b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes, scale, 1);
  const c4_f2 c = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes, scale, 2), d = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes, scale, 3);
  v[0] = a[0], v[1] = a[1], v[2] = b[0], v[3] = b[1], v[4] = c[0], v[5] = c[1], v[6] = d[0], v[7] = d[1];
}

}  // namespace msda
