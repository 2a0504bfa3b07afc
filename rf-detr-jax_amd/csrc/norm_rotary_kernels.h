// norm_rotary_kernels.h — gfx950 device code for the norm of every head of queries and keys with the rotary
// positions in the same pass, and its gradients.
//
// A row x of D channels (one head of one token) becomes R [x r w], r = 1 / sqrt(mean x^2 + eps), with R the rotation
// of rotary_kernels.h by the token's positions. For the cotangent dy, with g = R^T dy and u = g w:
//   dw = sum over rows of g x r,   dx = r (u - x r^2 mean(u x)).
//
// What bounds it at many tokens is reading and writing the rows: once each, x and dy once each in the backward, which
// forms r again. A row belongs to LPR lanes of 32 bytes each, whose two 16-byte pieces are the partners of the
// rotation, so that the sums over a row are a few exchanges inside a wave and nothing waits for other waves. A
// workgroup forms the angles of its tokens once, in LDS (rotary_kernels.h), for all heads of queries and keys.
// The weights' gradients: a lane's unit of the row stays the same over all its rows, so it sums in registers; the
// workgroup adds its lanes and writes one row of partial sums, and a second kernel adds those in their order (no atomics).
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

#include "rotary_kernels.h"

namespace msda {

struct NormRotaryParams {
  const void* x[2];   // queries, keys
  const void* dy[2];  // backward: the cotangents
  void* y[2];         // the results; backward: the gradients of x, or null
  const void* w[2];   // [dim], or null: ones
  float* part;        // backward: [workgroups][2][dim] sums of the weights' gradients, or null
  const void* positions;
  int64_t xs[2][2], gs[2][2], ys[2][2];  // element strides (token, head)
  int64_t ps[2];
  int position_type, weight_type;  // enum msda_position_type, enum msda_dtype
  int tokens, heads[2], dim, pairs;
  int per;            // tokens of a step of a workgroup
  float eps, inverse_dim;
  double turns[kRotMaxPairs];  // frequency / (2 pi)
  uint8_t axis[kRotMaxPairs];
};

// The cos and sin of `nt` tokens from t0 on, [nt][pairs] (as in rotary_kernel); SIGN -1: the rotation back.
template <int SIGN>
__device__ __forceinline__ void nr_angles(const NormRotaryParams& p, float2* cs, int64_t t0, int nt) {
  for (int i = threadIdx.x; i < nt * p.pairs; i += 256) {
    const int t = i / p.pairs, pair = i - t * p.pairs;
    const int64_t at = (t0 + t) * p.ps[0] + p.axis[pair] * p.ps[1];
    const double pos = p.position_type == 0   ? static_cast<double>(static_cast<const int32_t*>(p.positions)[at])
                       : p.position_type == 1 ? static_cast<double>(static_cast<const int64_t*>(p.positions)[at])
                                              : static_cast<double>(static_cast<const float*>(p.positions)[at]);
    const double turn = pos * p.turns[pair];
    float s, c;
    sincospif(2.0f * static_cast<float>(turn - rint(turn)), &s, &c);
    cs[i] = float2{c, SIGN * s};
  }
}

__device__ __forceinline__ float nr_weight(const NormRotaryParams& p, int which, int ch) {
  if (p.w[which] == nullptr) return 1.0f;
  return p.weight_type == 0 ? static_cast<const float*>(p.w[which])[ch] : rot_f32(static_cast<const bf16_t*>(p.w[which])[ch]);
}

template <int LPR>
__device__ __forceinline__ float nr_sum(float x) {
#pragma unroll
  for (int m = 1; m < LPR; m *= 2) x += __shfl_xor(x, m);
  return x;
}

// A lane's two pieces of a row, channels a .. a + E - 1 and b .. b + E - 1 (b < 0: none; a < 0: an idle lane).
template <typename T, bool NEIGHBOURS>
struct NrUnit {
  static constexpr int E = 16 / static_cast<int>(sizeof(T));
  int a, b;
  __device__ __forceinline__ NrUnit(const NormRotaryParams& p, int u) {
    if constexpr (NEIGHBOURS) {
      a = 2 * E * u;
    } else {
      const int turned = p.pairs / E;
      a = u < turned ? E * u : 2 * p.pairs + 2 * E * (u - turned);
      if (u < turned) {
        b = a + p.pairs;
        return;
      }
    }
    b = a + E < p.dim ? a + E : -1;
    if (a >= p.dim) a = b = -1;
  }
  __device__ __forceinline__ void load(const T* row, float* v) const {
#pragma unroll
    for (int j = 0; j < 2 * E; ++j) v[j] = 0.0f;
    if (a >= 0) rot_load<T>(v, row + a);
    if (b >= 0) rot_load<T>(v + E, row + b);
  }
  __device__ __forceinline__ void store(T* row, const float* v) const {
    if (a >= 0) rot_store<T>(row + a, v);
    if (b >= 0) rot_store<T>(row + b, v + E);
  }
  // cs: of the row's token
  __device__ __forceinline__ void turn(float* v, const float2* cs, int pairs) const {
    if constexpr (NEIGHBOURS) {
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const int ch = half == 0 ? a : b;
        if (ch < 0 || ch >= 2 * pairs) continue;
#pragma unroll
        for (int j = 0; j < E / 2; ++j) {
          const float2 f = cs[ch / 2 + j];
          const float s = v[half * E + 2 * j], t = v[half * E + 2 * j + 1];
          v[half * E + 2 * j] = s * f.x - t * f.y;
          v[half * E + 2 * j + 1] = s * f.y + t * f.x;
        }
      }
    } else {
      if (a < 0 || a >= pairs) return;
#pragma unroll
      for (int j = 0; j < E; ++j) {
        const float2 f = cs[a + j];
        const float s = v[j], t = v[E + j];
        v[j] = s * f.x - t * f.y;
        v[E + j] = s * f.y + t * f.x;
      }
    }
  }
  __device__ __forceinline__ void weights(const NormRotaryParams& p, int which, float* w) const {
#pragma unroll
    for (int j = 0; j < E; ++j) {
      w[j] = a >= 0 ? nr_weight(p, which, a + j) : 0.0f;
      w[E + j] = b >= 0 ? nr_weight(p, which, b + j) : 0.0f;
    }
  }
};

// Rows, their pieces and the rotation's halves on 16-byte boundaries.
template <typename T, int LPR, bool NEIGHBOURS>
__global__ void __launch_bounds__(256) norm_rotary_kernel(const NormRotaryParams p) {
  extern __shared__ __align__(16) float2 nr_cs[];  // [per][pairs]
  constexpr int E = 16 / static_cast<int>(sizeof(T)), SLOTS = 256 / LPR;
  const int64_t t0 = static_cast<int64_t>(blockIdx.x) * p.per;
  const int nt = static_cast<int>(min(static_cast<int64_t>(p.per), p.tokens - t0));
  const NrUnit<T, NEIGHBOURS> unit(p, static_cast<int>(threadIdx.x) % LPR);
  nr_angles<1>(p, nr_cs, t0, nt);
  __syncthreads();
#pragma unroll
  for (int which = 0; which < 2; ++which) {
    const int heads = p.heads[which];
    float w[2 * E], v[2 * E];
    unit.weights(p, which, w);
    for (int row = static_cast<int>(threadIdx.x) / LPR; row < nt * heads; row += SLOTS) {
      const int t = row / heads, h = row - t * heads;
      unit.load(static_cast<const T*>(p.x[which]) + (t0 + t) * p.xs[which][0] + h * p.xs[which][1], v);
      float sum = 0.0f;
#pragma unroll
      for (int j = 0; j < 2 * E; ++j) sum = fmaf(v[j], v[j], sum);
      const float r = rsqrtf(fmaf(nr_sum<LPR>(sum), p.inverse_dim, p.eps));
#pragma unroll
      for (int j = 0; j < 2 * E; ++j) v[j] *= r * w[j];
      unit.turn(v, nr_cs + t * p.pairs, p.pairs);
      unit.store(static_cast<T*>(p.y[which]) + (t0 + t) * p.ys[which][0] + h * p.ys[which][1], v);
    }
  }
}

// Queries, then keys: with the sums of both at a time 161 registers left 3 waves a SIMD (16,000 tokens of 40 heads, 128
// channels, bf16: 151 us, now 121 us).
template <typename T, int LPR, bool NEIGHBOURS>
__global__ void __launch_bounds__(256, 4) norm_rotary_bwd_kernel(const NormRotaryParams p) {
  extern __shared__ __align__(16) float2 nr_cs[];
  constexpr int E = 16 / static_cast<int>(sizeof(T)), SLOTS = 256 / LPR;
  __shared__ float sums[4][LPR][2 * E + 1];
  const int lane = static_cast<int>(threadIdx.x) & 63, wave = static_cast<int>(threadIdx.x) >> 6, u = lane % LPR;
  const NrUnit<T, NEIGHBOURS> unit(p, u);
  const int64_t stride = static_cast<int64_t>(gridDim.x) * p.per;
#pragma unroll 1
  for (int which = 0; which < 2; ++which) {
    const int heads = p.heads[which];
    float w[2 * E], dw[2 * E] = {};
    unit.weights(p, which, w);
    for (int64_t t0 = static_cast<int64_t>(blockIdx.x) * p.per; t0 < p.tokens; t0 += stride) {
      const int nt = static_cast<int>(min(static_cast<int64_t>(p.per), p.tokens - t0));
      if (which == 0 || stride < p.tokens) {  // (one step: they are there)
        __syncthreads();                       // the last step's angles are read
        nr_angles<-1>(p, nr_cs, t0, nt);
        __syncthreads();
      }
      const T* px = static_cast<const T*>(p.x[which]) + t0 * p.xs[which][0];
      const T* pg = static_cast<const T*>(p.dy[which]) + t0 * p.gs[which][0];
      T* py = static_cast<T*>(p.y[which]);
      for (int row = static_cast<int>(threadIdx.x) / LPR; row < nt * heads; row += SLOTS) {
        const int t = row / heads, h = row - t * heads;
        float x[2 * E], g[2 * E];
        unit.load(px + t * p.xs[which][0] + h * p.xs[which][1], x);
        unit.load(pg + t * p.gs[which][0] + h * p.gs[which][1], g);
        unit.turn(g, nr_cs + t * p.pairs, p.pairs);
        float xx = 0.0f, ux = 0.0f;
#pragma unroll
        for (int j = 0; j < 2 * E; ++j) {
          xx = fmaf(x[j], x[j], xx);
          ux = fmaf(g[j] * w[j], x[j], ux);
        }
        xx = nr_sum<LPR>(xx);
        ux = nr_sum<LPR>(ux);
        const float r = rsqrtf(fmaf(xx, p.inverse_dim, p.eps)), back = r * r * (ux * p.inverse_dim);
#pragma unroll
        for (int j = 0; j < 2 * E; ++j) {
          dw[j] = fmaf(g[j], x[j] * r, dw[j]);
          x[j] = r * fmaf(-x[j], back, g[j] * w[j]);
        }
        if (py != nullptr) unit.store(py + (t0 + t) * p.ys[which][0] + h * p.ys[which][1], x);
      }
    }
    if (p.part == nullptr) continue;
    __syncthreads();
#pragma unroll
    for (int j = 0; j < 2 * E; ++j) {
      float s = dw[j];
#pragma unroll
      for (int m = LPR; m < 64; m *= 2) s += __shfl_xor(s, m);
      if (lane < LPR) sums[wave][u][j] = s;
    }
    __syncthreads();
    for (int i = threadIdx.x; i < LPR * 2 * E; i += 256) {
      const int v = i / (2 * E), j = i - v * 2 * E;
      const NrUnit<T, NEIGHBOURS> of(p, v);
      const int ch = j < E ? (of.a < 0 ? -1 : of.a + j) : (of.b < 0 ? -1 : of.b + j - E);
      if (ch >= 0) p.part[(static_cast<int64_t>(blockIdx.x) * 2 + which) * p.dim + ch] = sums[0][v][j] + sums[1][v][j] + sums[2][v][j] + sums[3][v][j];
    }
  }
}

// Any sizes, strides and alignment: a wave takes a row, a lane the channels lane, lane + 64, ... and loads the other
// channel of each pair beside its own.
template <typename T, bool NEIGHBOURS, bool BACKWARD>
__global__ void __launch_bounds__(256) norm_rotary_any_kernel(const NormRotaryParams p) {
  extern __shared__ __align__(16) float2 nr_cs[];
  __shared__ float sums[4][2 * kRotMaxPairs];
  constexpr int N = 2 * kRotMaxPairs / 64;
  const int lane = static_cast<int>(threadIdx.x) & 63, wave = static_cast<int>(threadIdx.x) >> 6;
  float dw[2][N] = {};
  for (int64_t t0 = static_cast<int64_t>(blockIdx.x) * p.per; t0 < p.tokens; t0 += static_cast<int64_t>(gridDim.x) * p.per) {
    const int nt = static_cast<int>(min(static_cast<int64_t>(p.per), p.tokens - t0));
    __syncthreads();
    nr_angles<BACKWARD ? -1 : 1>(p, nr_cs, t0, nt);
    __syncthreads();
#pragma unroll
    for (int which = 0; which < 2; ++which) {
      const int heads = p.heads[which];
      for (int row = wave; row < nt * heads; row += 4) {
        const int t = row / heads, h = row - t * heads;
        const T* x = static_cast<const T*>(p.x[which]) + (t0 + t) * p.xs[which][0] + h * p.xs[which][1];
        const T* dy = BACKWARD ? static_cast<const T*>(p.dy[which]) + (t0 + t) * p.gs[which][0] + h * p.gs[which][1] : nullptr;
        T* y = static_cast<T*>(p.y[which]) + (p.y[which] != nullptr ? (t0 + t) * p.ys[which][0] + h * p.ys[which][1] : 0);
        float v[N], w[N], to[N], xx = 0.0f, ux = 0.0f;  // forward: `to` is the other channel, normed; backward: g
#pragma unroll
        for (int j = 0; j < N; ++j) {
          const int ch = lane + 64 * j;
          v[j] = w[j] = to[j] = 0.0f;
          if (ch >= p.dim) continue;
          v[j] = rot_f32(x[ch]);
          w[j] = nr_weight(p, which, ch);
          xx = fmaf(v[j], v[j], xx);
          const bool turned = ch < 2 * p.pairs, first = NEIGHBOURS ? ch % 2 == 0 : ch < p.pairs;
          const int pair = NEIGHBOURS ? ch / 2 : first ? ch : ch - p.pairs, other = NEIGHBOURS ? ch ^ 1 : first ? ch + p.pairs : ch - p.pairs;
          if constexpr (BACKWARD) {
            to[j] = rot_f32(dy[ch]);
            if (turned) {
              const float2 f = nr_cs[t * p.pairs + pair];
              const float o = rot_f32(dy[other]);
              to[j] = first ? to[j] * f.x - o * f.y : to[j] * f.x + o * f.y;
            }
            ux = fmaf(to[j] * w[j], v[j], ux);
          } else if (turned) {
            to[j] = rot_f32(x[other]) * nr_weight(p, which, other);
          }
        }
        const float r = rsqrtf(fmaf(nr_sum<64>(xx), p.inverse_dim, p.eps));
        const float back = BACKWARD ? r * r * (nr_sum<64>(ux) * p.inverse_dim) : 0.0f;
#pragma unroll
        for (int j = 0; j < N; ++j) {
          const int ch = lane + 64 * j;
          if (ch >= p.dim) continue;
          if constexpr (BACKWARD) {
            dw[which][j] = fmaf(to[j], v[j] * r, dw[which][j]);
            if (p.y[which] != nullptr) rot_put(y[ch], r * fmaf(-v[j], back, to[j] * w[j]));
          } else {
            const bool turned = ch < 2 * p.pairs, first = NEIGHBOURS ? ch % 2 == 0 : ch < p.pairs;
            float z = v[j] * w[j] * r;
            if (turned) {
              const float2 f = nr_cs[t * p.pairs + (NEIGHBOURS ? ch / 2 : first ? ch : ch - p.pairs)];
              const float o = to[j] * r;
              z = first ? z * f.x - o * f.y : o * f.y + z * f.x;
            }
            rot_put(y[ch], z);
          }
        }
      }
    }
  }
  if (!BACKWARD || p.part == nullptr) return;
#pragma unroll
  for (int which = 0; which < 2; ++which) {
    __syncthreads();
#pragma unroll
    for (int j = 0; j < N; ++j) sums[wave][lane + 64 * j] = dw[which][j];
    __syncthreads();
    for (int ch = threadIdx.x; ch < p.dim; ch += 256)
      p.part[(static_cast<int64_t>(blockIdx.x) * 2 + which) * p.dim + ch] = sums[0][ch] + sums[1][ch] + sums[2][ch] + sums[3][ch];
  }
}

// The workgroups' sums of the weights' gradients, in their order: 16 columns of [2][dim] to a workgroup, 4 to a thread.
__global__ void __launch_bounds__(1024) norm_rotary_join_kernel(const float* part, int rows, int dim, void* q, void* k, int weight_type) {
  __shared__ float sums[256][17];
  const int quad = static_cast<int>(threadIdx.x) & 3, at = static_cast<int>(threadIdx.x) >> 2, c = static_cast<int>(blockIdx.x) * 16 + 4 * quad;
  float4 s = {0.0f, 0.0f, 0.0f, 0.0f};
  if (c < 2 * dim) {  // (2 dim is a multiple of 4)
#pragma unroll 4
    for (int r = at; r < rows; r += 256) {
      const float4 x = *reinterpret_cast<const float4*>(part + static_cast<int64_t>(r) * 2 * dim + c);
      s.x += x.x, s.y += x.y, s.z += x.z, s.w += x.w;
    }
  }
  sums[at][4 * quad] = s.x, sums[at][4 * quad + 1] = s.y, sums[at][4 * quad + 2] = s.z, sums[at][4 * quad + 3] = s.w;
  __syncthreads();
  // 16 columns of 64 threads each
  const int col = static_cast<int>(threadIdx.x) & 15, row = static_cast<int>(threadIdx.x) >> 4, to_col = static_cast<int>(blockIdx.x) * 16 + col;
  float t = (sums[row][col] + sums[row + 64][col]) + (sums[row + 128][col] + sums[row + 192][col]);
  __syncthreads();
  sums[row][col] = t;
  __syncthreads();
  for (int n = 32; n > 0; n /= 2) {
    if (row < n) sums[row][col] += sums[row + n][col];
    __syncthreads();
  }
  if (row != 0 || to_col >= 2 * dim) return;
  void* to = to_col < dim ? q : k;
  const int ch = to_col < dim ? to_col : to_col - dim;
  if (to == nullptr) return;
  if (weight_type == 0) static_cast<float*>(to)[ch] = sums[0][col];
  else rot_put(static_cast<bf16_t*>(to)[ch], sums[0][col]);
}

}  // namespace msda
