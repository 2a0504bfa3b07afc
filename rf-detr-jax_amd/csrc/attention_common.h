// attention_common.h — what the attention kernels share: register types, the softmax's exponential,
// reductions over a wave's halves, bf16 operands and transposing LDS reads.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

namespace msda {

typedef float at_f4 __attribute__((ext_vector_type(4)));
typedef float at_f16 __attribute__((ext_vector_type(16)));
typedef __bf16 at_bf8 __attribute__((ext_vector_type(8)));
typedef float at_f8 __attribute__((ext_vector_type(8)));

__device__ __forceinline__ at_bf8 at_bf8_of(uint2 lo, uint2 hi) { return __builtin_bit_cast(at_bf8, uint4{lo.x, lo.y, hi.x, hi.y}); }

// registers i0 .. i0 + 7 of a result block, rounded to bf16 (v_cvt_pk_bf16_f32, nearest even)
__device__ __forceinline__ at_bf8 at_bf8_regs(const at_f16& v, int i0) {
  const at_f8 f = {v[i0], v[i0 + 1], v[i0 + 2], v[i0 + 3], v[i0 + 4], v[i0 + 5], v[i0 + 6], v[i0 + 7]};
  return __builtin_convertvector(f, at_bf8);
}

// 2^x by v_exp_f32 alone: results below 2^-126 flush to zero (a weight that small is below the
// f32 resolution of any row sum it enters), 2^-inf = 0.
__device__ __forceinline__ float at_exp2(float x) { return __builtin_amdgcn_exp2f(x); }

__device__ __forceinline__ at_f16 at_zero16() {
  at_f16 z;
#pragma unroll
  for (int i = 0; i < 16; ++i) z[i] = 0.0f;
  return z;
}

// Reductions over the two halves of a wave (lanes l and l ^ 32, which hold the same query) by
// v_permlane32_swap: both lanes get the same bits.
__device__ __forceinline__ float at_max_halves(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}

__device__ __forceinline__ float at_sum_halves(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// A running reference score moves only when a chunk's maximum exceeds it by more than kAtLazy, or, while
// nothing has been summed, lies more than kAtLow below it (both log2): weights stay within 2^kAtLazy,
// which f32 sums and bf16 operands hold as well as weights within 1.
constexpr float kAtLazy = 8.0f;
constexpr float kAtLow = 64.0f;

typedef short at_s4 __attribute__((ext_vector_type(4)));

// ds_read_b64_tr_b16: within each group of 16 lanes, lane 4a + b receives element b of the 8 bytes
// that lanes a, 4 + a, 8 + a and 12 + a address (in that order): the 16 x 4 block of 16-bit
// elements the group addresses, transposed.
__device__ __forceinline__ uint2 at_read_tr(const uint16_t* p) {
  const at_s4 r = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) at_s4*)(p));
  return __builtin_bit_cast(uint2, r);
}

}  // namespace msda
