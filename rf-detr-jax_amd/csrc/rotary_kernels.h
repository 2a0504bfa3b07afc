// rotary_kernels.h — gfx950 device code for rotary positions on several axes, of queries and keys in one
// launch.
//
// Channel pair i of a head belongs to one axis a and has a frequency f; with the token's position x_a on
// that axis, the pair (u, w) becomes (u cos - w sin, u sin + w cos) of the angle x_a f. The gradient is
// the same rotation by -angle. Channels behind the pairs pass unchanged.
//
// Angles. A position of 10^6 leaves no fraction of a turn in f32 at a frequency of 1, so the angle is
// formed in turns in f64, its whole turns dropped, and only then rounded: cos and sin are those of f32
// arguments in [-1/2, 1/2] turns whatever the position. They cost far more than the two products of a
// pair, and every head of a token uses the same: a workgroup forms them once per (token, pair) in LDS
// and then streams the rows of all heads, 32 bytes a thread and step. What bounds the kernel at many
// tokens is reading and writing the rows.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

#include "msda_kernels.h"  // bf16_t

namespace msda {

constexpr int kRotMaxPairs = 128;
constexpr int kRotMaxAxes = 8;

struct RotaryParams {
  const void* x[2];  // queries, keys
  void* y[2];
  const void* positions;
  int64_t xs[2][2], ys[2][2];  // element strides (token, head)
  int64_t ps[2];               // positions: element strides (token, axis)
  int position_type;           // enum msda_position_type
  int tokens, heads[2], dim, pairs;
  int per;                     // tokens of a workgroup
  float sign;                  // -1: the gradient
  double turns[kRotMaxPairs];  // frequency / (2 pi)
  uint8_t axis[kRotMaxPairs];
};

__device__ __forceinline__ float rot_f32(bf16_t v) { return __uint_as_float(static_cast<uint32_t>(v) << 16); }
__device__ __forceinline__ float rot_f32(float v) { return v; }
__device__ __forceinline__ void rot_put(bf16_t& y, float v) { y = __builtin_bit_cast(bf16_t, static_cast<__bf16>(v)); }  // nearest even
__device__ __forceinline__ void rot_put(float& y, float v) { y = v; }

// one 16-byte piece of a row
template <typename T>
__device__ __forceinline__ void rot_load(float* v, const T* x) {
  alignas(16) T e[16 / sizeof(T)];
  *reinterpret_cast<uint4*>(e) = *reinterpret_cast<const uint4*>(x);
#pragma unroll
  for (int j = 0; j < static_cast<int>(16 / sizeof(T)); ++j) v[j] = rot_f32(e[j]);
}
template <typename T>
__device__ __forceinline__ void rot_store(T* y, const float* v) {
  alignas(16) T e[16 / sizeof(T)];
#pragma unroll
  for (int j = 0; j < static_cast<int>(16 / sizeof(T)); ++j) rot_put(e[j], v[j]);
  *reinterpret_cast<uint4*>(y) = *reinterpret_cast<const uint4*>(e);
}

// VEC: pairs of a work item (their channels are two 16-byte pieces, or one where pairs are neighbours);
// 1: any sizes, strides and alignment, element by element.
template <typename T, int VEC, bool NEIGHBOURS>
__global__ void __launch_bounds__(256) rotary_kernel(const RotaryParams p) {
  extern __shared__ __align__(16) float2 rot_cs[];  // [per][pairs]: cos, sin
  const int64_t t0 = static_cast<int64_t>(blockIdx.x) * p.per;
  const int nt = static_cast<int>(min(static_cast<int64_t>(p.per), p.tokens - t0));
  for (int i = threadIdx.x; i < nt * p.pairs; i += 256) {
    const int t = i / p.pairs, pair = i - t * p.pairs;
    const int64_t at = (t0 + t) * p.ps[0] + p.axis[pair] * p.ps[1];
    const double pos = p.position_type == 0   ? static_cast<double>(static_cast<const int32_t*>(p.positions)[at])
                       : p.position_type == 1 ? static_cast<double>(static_cast<const int64_t*>(p.positions)[at])
                                              : static_cast<double>(static_cast<const float*>(p.positions)[at]);
    const double turn = pos * p.turns[pair];
    float s, c;
    sincospif(2.0f * static_cast<float>(turn - rint(turn)), &s, &c);
    rot_cs[i] = float2{c, s * p.sign};
  }
  __syncthreads();
  // items of a row: turned ones, then pieces that pass; rows of the workgroup: (token, head of q, then k)
  constexpr int E = VEC == 1 ? 1 : 16 / static_cast<int>(sizeof(T));
  const int turned = p.pairs / VEC, units = turned + (p.dim - 2 * p.pairs) / E, heads = p.heads[0] + p.heads[1];
  const int items = nt * heads * units;
  for (int i = threadIdx.x; i < items; i += 256) {
    const int row = i / units, u = i - row * units, t = row / heads;
    int h = row - t * heads;
    const int which = h >= p.heads[0] ? 1 : 0;
    if (which) h -= p.heads[0];
    const T* x = static_cast<const T*>(p.x[which]) + (t0 + t) * p.xs[which][0] + h * p.xs[which][1];
    T* y = static_cast<T*>(p.y[which]) + (t0 + t) * p.ys[which][0] + h * p.ys[which][1];
    if (u >= turned) {
      const int ch = 2 * p.pairs + (u - turned) * E;
      if constexpr (VEC == 1) y[ch] = x[ch];
      else *reinterpret_cast<uint4*>(y + ch) = *reinterpret_cast<const uint4*>(x + ch);
      continue;
    }
    const float2* cs = rot_cs + t * p.pairs + u * VEC;
    if constexpr (VEC == 1) {
      const int a = NEIGHBOURS ? 2 * u : u, b = NEIGHBOURS ? 2 * u + 1 : u + p.pairs;
      const float xa = rot_f32(x[a]), xb = rot_f32(x[b]);
      rot_put(y[a], xa * cs->x - xb * cs->y);
      rot_put(y[b], xa * cs->y + xb * cs->x);
    } else if constexpr (NEIGHBOURS) {
      float v[2 * VEC];
      rot_load<T>(v, x + 2 * VEC * u);
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        const float a = v[2 * j], b = v[2 * j + 1];
        v[2 * j] = a * cs[j].x - b * cs[j].y;
        v[2 * j + 1] = a * cs[j].y + b * cs[j].x;
      }
      rot_store<T>(y + 2 * VEC * u, v);
    } else {
      float a[VEC], b[VEC];
      rot_load<T>(a, x + VEC * u);
      rot_load<T>(b, x + VEC * u + p.pairs);
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        const float s = a[j], w = b[j];
        a[j] = s * cs[j].x - w * cs[j].y;
        b[j] = s * cs[j].y + w * cs[j].x;
      }
      rot_store<T>(y + VEC * u, a);
      rot_store<T>(y + VEC * u + p.pairs, b);
    }
  }
}

}  // namespace msda
