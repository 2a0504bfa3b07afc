// packed_attention_kernels.h — gfx950 device code for softmax attention over packed sequences of
// different lengths, with fewer key heads than query heads, causal or not, and its gradients.
//
// Sequence i has n queries, m keys and G = heads / kv_heads query heads to a key head:
//   s = scale q_t . k_j for the keys j < m (causal: j <= t + m - n), p = softmax_j(s), out_t = sum_j p v_j
// and out_t = 0 where no key is seen. Backward, with delta_t = do_t . out_t:
//   ds = p (do_t . v_j - delta_t), dq_t = scale sum_j ds k_j, dk_j = scale sum_t ds q_t, dv_j = sum_t p do_t,
// the sums over t also over the G query heads of the key head.
//
// Rows. The G query heads of one key head are read as rows of one matrix, r = t G + g, so that a tile of
// keys serves all of them, a new token of every head fills one tile, and dk and dv are summed over the
// heads inside one workgroup (no atomics, one order).
//
// Finding the tile. The tiles of BM rows lie in slots: segment s (the rows before the first sequence,
// the sequences, the rows behind the last) takes the slots from floor(first row / BM) + s on, which are
// at least ceil(rows / BM) many. So the grid is rows / BM + segments, known without the lengths, and a
// workgroup finds its segment by a search over the offsets alone: no length is read back by the host
// and no launch prepares a table. Offsets are clamped to the tensors' rows: wrong ones give wrong values
// and no access out of bounds. Rows outside every sequence are written as zeros.
//
// Layouts of the products as in attention_kernels.h: scores are formed transposed (streamed rows x own
// rows), a lane owns one own row (its softmax statistics stay in the lane), and the weights in their
// result registers are the B operand of the next product, whose A operand is read from the streamed
// tile by transposing LDS reads. Streamed tiles of 64 rows lie in LDS as swizzled rows, written by
// global_load_lds (no registers, two buffers, one barrier a tile); rows past a sequence's end and
// channels past head_dim come from a page of zeros.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

#include "attention_common.h"
#include "msda_kernels.h"  // bf16_t, wait_vmem

namespace msda {

enum PackTensor { kPkQ = 0, kPkK, kPkV, kPkO, kPkGO, kPkGQ, kPkGK, kPkGV, kPkTensors };

struct PackParams {
  const void* q;
  const void* k;
  const void* v;
  const void* o;   // backward: the forward output
  const void* go;  // backward: grad of the output
  void* out;
  void* gq;  // backward outputs (each may be null)
  void* gk;
  void* gv;
  float* stats;  // [q_rows * heads][4]: m, log2 l (forward), delta (backward), unused; row (token, head)
  const int32_t* q_offsets;  // [sequences + 1]
  const int32_t* k_offsets;  // [sequences + 1]
  const int32_t* k_lengths;  // [sequences], or null: all rows of a sequence's range
  float* part_o;             // split forward: [splits][q_rows * heads][dim], sums relative to part_ml's m
  float* part_ml;            // [splits][q_rows * heads][2]: m, l
  int64_t st[kPkTensors][2];  // element strides (row, head) of each tensor
  int sequences, q_rows, k_rows, heads, kv_heads, group, dim, causal, splits;
  int slots;     // tiles of the kernel's own side
  float scale;   // of the scores
  float scale2;  // scale log2(e)
};

constexpr int kPkTile = 128;  // own rows of a workgroup: 32 a wave
constexpr int kPkChunk = 64;  // streamed rows of a tile

__device__ __align__(16) const uint32_t pk_zeros[4] = {0u, 0u, 0u, 0u};

// ---- the workgroup's place ---------------------------------------------------------------------

// First row of segment s, 0 <= s <= sequences + 2, clamped to the tensor.
__device__ __forceinline__ int pk_bound(const int32_t* offsets, int s, int sequences, int rows) {
  if (s == 0) return 0;
  if (s >= sequences + 2) return rows;
  return min(max(offsets[s - 1], 0), rows);
}

struct PkPlace {
  int seq;         // the sequence, or -1: rows outside every sequence
  int first;       // first row of the segment in the own tensor
  int own;         // its rows (tokens)
  int tile;        // tile of the segment
};

// The segment of `slot` (the wave searches 64 segments at a time): the last one that starts at or
// before it. `unit`: rows of a tile's matrix to a row of the tensor.
template <int BM>
__device__ __forceinline__ PkPlace pk_place(const int32_t* offsets, int sequences, int rows, int unit, int slot, int lane) {
  int lo = 0, hi = sequences + 2;
  while (hi - lo > 1) {
    const int step = (hi - lo + 63) / 64, s = lo + lane * step;
    const bool at = s < hi && static_cast<int>(static_cast<uint32_t>(pk_bound(offsets, s, sequences, rows)) * unit / BM) + s <= slot;
    const int n = max(1, static_cast<int>(__popcll(__ballot(at))));
    lo += (n - 1) * step;
    hi = min(hi, lo + step);
  }
  lo = __builtin_amdgcn_readfirstlane(lo);
  PkPlace w;
  w.first = pk_bound(offsets, lo, sequences, rows);
  w.own = max(0, pk_bound(offsets, lo + 1, sequences, rows) - w.first);
  w.seq = lo >= 1 && lo <= sequences ? lo - 1 : -1;
  w.tile = slot - (static_cast<int>(static_cast<uint32_t>(w.first) * unit / BM) + lo);
  if (w.tile < 0) w.tile = w.own = 0;  // only where the offsets fall
  return w;
}

// ---- operands ----------------------------------------------------------------------------------

// DT: channels that the products run over (head_dim rounded up to 32); a tile's rows lie DP apart.
template <typename T, int DT>
struct PkTile {
  static constexpr int DP = DT == 96 ? 128 : DT;
  static constexpr int E = 16 / static_cast<int>(sizeof(T));  // elements of a 16-byte chunk
  static constexpr int CPR = DP / E;                          // chunks of a row
  static constexpr int BYTES = kPkChunk * DP * static_cast<int>(sizeof(T));
  static constexpr int ND = DT / 32;
  // 16-byte chunk c of row r sits at slot c ^ swizzle(r): the rows that a read takes together fall on
  // distinct banks
  static __device__ __forceinline__ int swizzle(int r) { return CPR >= 16 ? (r & 15) : ((r / (16 / CPR)) & (CPR - 1)); }
  static __device__ __forceinline__ int at(int r, int ch) { return r * DP + E * ((ch / E) ^ swizzle(r)) + (ch % E); }
};

// One row's channels as the B operand of the score products.
template <typename T, int DT>
struct PkRow;
template <int DT>
struct PkRow<bf16_t, DT> {
  at_bf8 x[DT / 16];  // channels 16 s + 8 grp .. + 7
  __device__ __forceinline__ void load(const bf16_t* row, bool valid, int dim, int grp) {
#pragma unroll
    for (int s = 0; s < DT / 16; ++s) {
      const int ch = 16 * s + 8 * grp;
      const void* p = valid && ch < dim ? static_cast<const void*>(reinterpret_cast<const uint16_t*>(row) + ch) : static_cast<const void*>(pk_zeros);
      x[s] = __builtin_bit_cast(at_bf8, *static_cast<const uint4*>(p));
    }
  }
  __device__ __forceinline__ float dot(const PkRow& y) const {  // this half-wave's channels
    float d = 0.0f;
#pragma unroll
    for (int s = 0; s < DT / 16; ++s) {
      const at_f8 a = __builtin_convertvector(x[s], at_f8), b = __builtin_convertvector(y.x[s], at_f8);
#pragma unroll
      for (int j = 0; j < 8; ++j) d = fmaf(a[j], b[j], d);
    }
    return d;
  }
};
template <int DT>
struct PkRow<float, DT> {
  at_f4 x[DT / 8];  // channels 8 c + 4 grp .. + 3
  __device__ __forceinline__ void load(const float* row, bool valid, int dim, int grp) {
#pragma unroll
    for (int c = 0; c < DT / 8; ++c) {
      const int ch = 8 * c + 4 * grp;
      const void* p = valid && ch < dim ? static_cast<const void*>(row + ch) : static_cast<const void*>(pk_zeros);
      x[c] = *static_cast<const at_f4*>(p);
    }
  }
  __device__ __forceinline__ float dot(const PkRow& y) const {
    float d = 0.0f;
#pragma unroll
    for (int c = 0; c < DT / 8; ++c)
#pragma unroll
      for (int j = 0; j < 4; ++j) d = fmaf(x[c][j], y.x[c][j], d);
    return d;
  }
};

// Scores of the 32-row block at row x0 of a tile against the lane's row: register i holds streamed row
// x0 + 8 (i / 4) + 4 grp + i % 4.
template <typename T, int DT>
__device__ __forceinline__ at_f16 pk_scores(const T* X, int x0, const PkRow<T, DT>& r, int col, int grp) {
  using Tile = PkTile<T, DT>;
  at_f16 s = at_zero16();
  if constexpr (sizeof(T) == 2) {
#pragma unroll
    for (int i = 0; i < DT / 16; ++i) {
      const at_bf8 a = __builtin_bit_cast(at_bf8, *reinterpret_cast<const uint4*>(&X[Tile::at(x0 + col, 16 * i + 8 * grp)]));
      s = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, r.x[i], s, 0, 0, 0);
    }
  } else {
#pragma unroll
    for (int c = 0; c < DT / 8; ++c) {
      const at_f4 a = *reinterpret_cast<const at_f4*>(&X[Tile::at(x0 + col, 8 * c + 4 * grp)]);
#pragma unroll
      for (int j = 0; j < 4; ++j) s = __builtin_amdgcn_mfma_f32_32x32x2f32(a[j], r.x[c][j], s, 0, 0, 0);
    }
  }
  return s;
}

// acc += X^T w for the 32-row block at row x0 of a tile, w in result-layout registers: acc[nd] register i
// holds channel 32 nd + 8 (i / 4) + 4 grp + i % 4 of the lane's row. bf16: w is rounded to bf16 for the
// product (half a step, 2^-8 of each weight at most: as much as the inputs' and the result's own rounding).
template <typename T, int DT>
__device__ __forceinline__ void pk_accumulate(at_f16 (&acc)[DT / 32], const T* X, int x0, const at_f16& w, int lane) {
  using Tile = PkTile<T, DT>;
  const int grp = lane >> 5;
  if constexpr (sizeof(T) == 2) {
    const int g = lane >> 4, r = lane & 15;
    const uint16_t* U = reinterpret_cast<const uint16_t*>(X);
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      const at_bf8 b = at_bf8_regs(w, 8 * s);
#pragma unroll
      for (int nd = 0; nd < DT / 32; ++nd) {
        const int c = 32 * nd + 16 * (g & 1) + 4 * (r & 3), ro = x0 + 16 * s + 4 * grp + (r >> 2);
        const at_bf8 a = at_bf8_of(at_read_tr(U + Tile::at(ro, c)), at_read_tr(U + Tile::at(ro + 8, c)));
        acc[nd] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, acc[nd], 0, 0, 0);
      }
    }
  } else {
    const int col = lane & 31;
#pragma unroll
    for (int i = 0; i < 16; ++i)
#pragma unroll
      for (int nd = 0; nd < DT / 32; ++nd)
        acc[nd] = __builtin_amdgcn_mfma_f32_32x32x2f32(X[Tile::at(x0 + 8 * (i >> 2) + 4 * grp + (i & 3), 32 * nd + col)], w[i], acc[nd], 0, 0, 0);
  }
}

// A wave's LDS accesses are in order; this keeps the compiler from exchanging them.
__device__ __forceinline__ void pk_wave_sync() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// Writes acc * f (f: of the lane's row) as rows of T: through the wave's LDS scratch, so that each lane
// stores 16 bytes and the wave whole rows. `row(r)`: the address of own row r of the wave's 32, or null.
template <typename T, int DT, typename R>
__device__ __forceinline__ void pk_store(const at_f16 (&acc)[DT / 32], float f, T* scratch, int dim, int lane, R&& row) {
  constexpr int E = 16 / static_cast<int>(sizeof(T)), LD = DT + E, C = DT / E;
  static_assert(32 * LD * sizeof(T) <= PkTile<T, DT>::BYTES, "the scratch fits a tile");
  const int grp = lane >> 5, col = lane & 31;
#pragma unroll
  for (int nd = 0; nd < DT / 32; ++nd) {
    const at_f16 v = acc[nd] * f;
    if constexpr (sizeof(T) == 2) {
      uint16_t* t = reinterpret_cast<uint16_t*>(scratch) + col * LD + 32 * nd + 4 * grp;
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        const uint4 u = __builtin_bit_cast(uint4, at_bf8_regs(v, 8 * s));
        *reinterpret_cast<uint2*>(t + 16 * s) = uint2{u.x, u.y};
        *reinterpret_cast<uint2*>(t + 16 * s + 8) = uint2{u.z, u.w};
      }
    } else {
      float* t = scratch + col * LD + 32 * nd + 4 * grp;
#pragma unroll
      for (int c = 0; c < 4; ++c) *reinterpret_cast<at_f4*>(t + 8 * c) = at_f4{v[4 * c], v[4 * c + 1], v[4 * c + 2], v[4 * c + 3]};
    }
  }
  pk_wave_sync();
#pragma unroll
  for (int k = 0; k < C / 2; ++k) {
    const int idx = lane + 64 * k, r = idx / C, ch = E * (idx - r * C);
    T* to = row(r);
    if (to != nullptr && ch < dim) *reinterpret_cast<uint4*>(to + ch) = *reinterpret_cast<const uint4*>(scratch + r * LD + ch);
  }
  pk_wave_sync();
}

// Rows of zeros: own rows [r0, r1) of the matrix, `row(r)` their addresses, by the whole workgroup.
template <typename T, int NT, typename R>
__device__ __forceinline__ void pk_zero_rows(int r0, int r1, int dim, R&& row) {
  constexpr int E = 16 / static_cast<int>(sizeof(T));
  const int c = dim / E;
  for (int idx = threadIdx.x; idx < (r1 - r0) * c; idx += NT) {
    const int r = idx / c;
    *reinterpret_cast<uint4*>(row(r0 + r) + E * (idx - r * c)) = uint4{0u, 0u, 0u, 0u};
  }
}

// ---- streaming ---------------------------------------------------------------------------------

// The transfers of one 64-row tile by the workgroup's 256 threads: piece u is row u / CPR, slot u % CPR,
// which holds the row's chunk slot ^ swizzle(row).
template <typename T, int DT>
struct PkStream {
  using Tile = PkTile<T, DT>;
  static constexpr int NV = kPkChunk * Tile::CPR / 256;  // pieces of a thread
  // rows [first, first + 64) of a tensor whose row r is base + r stride; rows from `end` on are zeros
  static __device__ __forceinline__ void load(unsigned char* lds, const T* base, int64_t stride, int first, int end, int dim) {
    const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x >> 6));
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      const int u = threadIdx.x + 256 * v, row = u / Tile::CPR, ch = Tile::E * ((u % Tile::CPR) ^ Tile::swizzle(row));
      const void* src = first + row < end && ch < dim ? static_cast<const void*>(base + (first + row) * stride + ch) : static_cast<const void*>(pk_zeros);
      __builtin_amdgcn_global_load_lds(static_cast<const uint4*>(src), (MSDA_LDS void*)(lds + (256 * v + 64 * wave) * 16), 16, 0, 0);
    }
  }
  // the same for rows r = t group + g of queries: row r at base + t stride + g head
  static __device__ __forceinline__ void load_rows(unsigned char* lds, const T* base, int64_t stride, int64_t head, int group, int first, int end,
                                                   int dim) {
    const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x >> 6));
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      const int u = threadIdx.x + 256 * v, row = u / Tile::CPR, ch = Tile::E * ((u % Tile::CPR) ^ Tile::swizzle(row));
      const int r = first + row, t = r / group, g = r - t * group;
      const void* src = r < end && ch < dim ? static_cast<const void*>(base + t * stride + g * head + ch) : static_cast<const void*>(pk_zeros);
      __builtin_amdgcn_global_load_lds(static_cast<const uint4*>(src), (MSDA_LDS void*)(lds + (256 * v + 64 * wave) * 16), 16, 0, 0);
    }
  }
};

// ---- queries on their own side: forward and dq -------------------------------------------------

struct PkQueries {
  PkPlace w;
  int kv_head;      // key head
  int split;
  int rows, r0;     // rows of the sequence's matrix, first of the workgroup's
  int64_t k_first;  // first key row
  int m, shift;     // keys; a row of token t sees the keys below min(m, t + shift + 1)
  __device__ PkQueries(const PackParams& p, int lane) {
    // key heads fastest: with 8 of them each stays on one XCD, whose L2 then holds its keys; the last
    // tiles, which see the most keys of a causal sequence, first
    const int b = static_cast<int>(blockIdx.x), rest = b / p.kv_heads;
    kv_head = b - rest * p.kv_heads;
    const int slot = p.slots - 1 - rest / p.splits;
    split = rest % p.splits;
    w = pk_place<kPkTile>(p.q_offsets, p.sequences, p.q_rows, p.group, slot, lane);
    rows = w.own * p.group;
    r0 = w.tile * kPkTile;
    k_first = 0;
    m = 0;
    if (w.seq >= 0) {
      const int a = min(max(p.k_offsets[w.seq], 0), p.k_rows), b2 = min(max(p.k_offsets[w.seq + 1], a), p.k_rows);
      k_first = a;
      m = p.k_lengths != nullptr ? min(max(p.k_lengths[w.seq], 0), b2 - a) : b2 - a;
    }
    shift = m - w.own;
  }
  __device__ int seen(const PackParams& p, int r) const { return p.causal ? min(max(r / p.group + shift + 1, 0), m) : m; }
  template <typename T>
  __device__ T* row(const PackParams& p, T* base, int t, int r) const {
    const int tok = r / p.group, g = r - tok * p.group;
    return base + (w.first + tok) * p.st[t][0] + (kv_head * p.group + g) * p.st[t][1];
  }
  __device__ int64_t stat(const PackParams& p, int r) const {
    const int tok = r / p.group, g = r - tok * p.group;
    return static_cast<int64_t>(w.first + tok) * p.heads + kv_head * p.group + g;
  }
};

// The statistics of a row: m and log2 l as two numbers whose sum the backward subtracts without rounding
// it at its own size. With l = 2^e f, f in [1, 2): m + e, and log2 f with what that sum rounds off. A row
// that saw no key: every weight is 2^-inf.
__device__ __forceinline__ float2 pk_stats(float m, float l) {
  if (l == 0.0f) return float2{0.0f, INFINITY};
  const float e = static_cast<float>(static_cast<int>(__float_as_uint(l) >> 23) - 127);
  const float f = __uint_as_float((__float_as_uint(l) & 0x007fffffu) | 0x3f800000u);
  const float me = m + e, t = me - m;
  return float2{me, l - l == 0.0f ? log2f(f) + ((m - (me - t)) + (e - t)) : l};  // an l that is no number stays one
}

// Scores of keys from `lim` on become -inf (register i: key k0 + 8 (i / 4) + 4 grp + i % 4).
__device__ __forceinline__ void pk_mask(at_f16& s, int k0, int lim, int grp) {
#pragma unroll
  for (int i = 0; i < 16; ++i) s[i] = k0 + 8 * (i >> 2) + 4 * grp + (i & 3) < lim ? s[i] : -INFINITY;
}

// Forward. A workgroup takes 128 rows and walks over the keys that they see, 64 at a time, with a running
// reference score m (moved when a chunk's maximum exceeds it by 2^8, or lies 2^64 below it while nothing
// is summed) and sum l.
template <typename T, int DT>
__global__ void __launch_bounds__(256, sizeof(T) == 2 ? 2 : 1) pk_fwd_kernel(const PackParams p) {
  using Tile = PkTile<T, DT>;
  __shared__ __align__(16) unsigned char K0[Tile::BYTES], V0[Tile::BYTES], K1[Tile::BYTES], V1[Tile::BYTES];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, grp = lane >> 5, col = lane & 31;
  const PkQueries w(p, lane);
  if (w.r0 >= w.rows) return;
  const int r1 = min(w.r0 + kPkTile, w.rows);
  T* out = static_cast<T*>(p.out);
  if (w.w.seq < 0) {
    if (p.splits == 1) {
      pk_zero_rows<T, 256>(w.r0, r1, p.dim, [&](int r) { return w.row(p, out, kPkO, r); });
    } else {
      for (int r = w.r0 + static_cast<int>(threadIdx.x); r < r1; r += 256)
        *reinterpret_cast<float2*>(p.part_ml + (static_cast<int64_t>(w.split) * p.q_rows * p.heads + w.stat(p, r)) * 2) = float2{0.0f, 0.0f};
    }
    return;
  }
  const int wr0 = w.r0 + 32 * wave, ri = wr0 + col;
  const bool valid = ri < w.rows;
  const int lim = valid ? w.seen(p, ri) : 0;
  const int end = w.seen(p, r1 - 1);                                          // keys that the workgroup sees
  const int wend = wr0 < w.rows ? w.seen(p, min(wr0 + 31, w.rows - 1)) : 0;   // the wave
  const int wfull = wr0 + 31 < w.rows ? w.seen(p, wr0) : 0;                   // every row of the wave
  int c0 = 0, c1 = (end + kPkChunk - 1) / kPkChunk;
  if (p.splits > 1) {
    const int per = (c1 + p.splits - 1) / p.splits;
    c0 = min(c1, w.split * per);
    c1 = min(c1, c0 + per);
  }
  PkRow<T, DT> q;
  q.load(w.row(p, static_cast<const T*>(p.q), kPkQ, min(ri, w.rows - 1)), valid, p.dim, grp);
  const T* kp = static_cast<const T*>(p.k) + w.k_first * p.st[kPkK][0] + w.kv_head * p.st[kPkK][1];
  const T* vp = static_cast<const T*>(p.v) + w.k_first * p.st[kPkV][0] + w.kv_head * p.st[kPkV][1];
  float m = 0.0f, l = 0.0f;
  at_f16 o[DT / 32];
#pragma unroll
  for (int nd = 0; nd < DT / 32; ++nd) o[nd] = at_zero16();

  auto stage = [&](unsigned char* K, unsigned char* V, int c) {
    PkStream<T, DT>::load(K, kp, p.st[kPkK][0], c * kPkChunk, w.m, p.dim);
    PkStream<T, DT>::load(V, vp, p.st[kPkV][0], c * kPkChunk, w.m, p.dim);
  };
  auto chunk = [&](const unsigned char* Kb, const unsigned char* Vb, int c) {
    const T* K = reinterpret_cast<const T*>(Kb);
    const T* V = reinterpret_cast<const T*>(Vb);
    const int k0 = c * kPkChunk;
    if (k0 >= wend) return;
    at_f16 s0 = pk_scores<T, DT>(K, 0, q, col, grp), s1 = pk_scores<T, DT>(K, 32, q, col, grp);
    if (k0 + kPkChunk > wfull) {
      pk_mask(s0, k0, lim, grp);
      pk_mask(s1, k0 + 32, lim, grp);
    }
    float bm = -INFINITY;
#pragma unroll
    for (int i = 0; i < 16; ++i) bm = fmaxf(bm, fmaxf(s0[i], s1[i]));
    bm = at_max_halves(bm) * p.scale2;
    if (bm != -INFINITY && (bm > m + kAtLazy || (l == 0.0f && bm < m - kAtLow))) {
      const float alpha = l == 0.0f ? 0.0f : at_exp2(m - bm);
      m = bm;
      l *= alpha;
#pragma unroll
      for (int nd = 0; nd < DT / 32; ++nd) o[nd] *= alpha;
    }
    float rs = 0.0f;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      s0[i] = at_exp2(fmaf(s0[i], p.scale2, -m));
      s1[i] = at_exp2(fmaf(s1[i], p.scale2, -m));
      rs += s0[i] + s1[i];
    }
    l += at_sum_halves(rs);
    pk_accumulate<T, DT>(o, V, 0, s0, lane);
    pk_accumulate<T, DT>(o, V, 32, s1, lane);
  };
  if (c0 < c1) stage(K0, V0, c0);
  for (int c = c0; c < c1; c += 2) {
    wait_vmem();
    __syncthreads();  // tile c is there, and every wave is done with tile c - 1
    if (c + 1 < c1) stage(K1, V1, c + 1);
    chunk(K0, V0, c);
    if (c + 1 >= c1) break;
    wait_vmem();
    __syncthreads();
    if (c + 2 < c1) stage(K0, V0, c + 2);
    chunk(K1, V1, c + 1);
  }
  __syncthreads();  // the tiles hold the waves' scratch from here
  unsigned char* const tiles[4] = {K0, V0, K1, V1};
  T* scratch = reinterpret_cast<T*>(wave == 0 ? tiles[0] : wave == 1 ? tiles[1] : wave == 2 ? tiles[2] : tiles[3]);
  if (p.splits > 1) {  // sums as they are: registers hold 4 consecutive channels of the lane's row
    if (!valid) return;
    const int64_t at = static_cast<int64_t>(w.split) * p.q_rows * p.heads + w.stat(p, ri);
    float* po = p.part_o + at * p.dim;
#pragma unroll
    for (int nd = 0; nd < DT / 32; ++nd)
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const int ch = 32 * nd + 8 * c + 4 * grp;
        if (ch < p.dim) *reinterpret_cast<at_f4*>(po + ch) = at_f4{o[nd][4 * c], o[nd][4 * c + 1], o[nd][4 * c + 2], o[nd][4 * c + 3]};
      }
    if (grp == 0) *reinterpret_cast<float2*>(p.part_ml + at * 2) = float2{m, l};
    return;
  }
  pk_store<T, DT>(o, l == 0.0f ? 0.0f : 1.0f / l, scratch, p.dim, lane,
                  [&](int r) { return wr0 + r < w.rows ? w.row(p, out, kPkO, wr0 + r) : static_cast<T*>(nullptr); });
  if (p.stats != nullptr && valid && grp == 0)
    *reinterpret_cast<float2*>(p.stats + 4 * w.stat(p, ri)) = pk_stats(m, l);
}

// The split forward's parts joined: one row (token, head) to a wave's quarter, 16 lanes a row.
template <typename T>
__global__ void __launch_bounds__(256) pk_join_kernel(const PackParams p) {
  const int64_t rows = static_cast<int64_t>(p.q_rows) * p.heads, row = static_cast<int64_t>(blockIdx.x) * 16 + (threadIdx.x >> 4);
  if (row >= rows) return;
  const int lane = threadIdx.x & 15;
  float m = -INFINITY, l = 0.0f;
  for (int s = 0; s < p.splits; ++s) {
    const float2 ml = *reinterpret_cast<const float2*>(p.part_ml + (s * rows + row) * 2);
    if (ml.y != 0.0f) m = fmaxf(m, ml.x);
  }
  for (int s = 0; s < p.splits; ++s) {
    const float2 ml = *reinterpret_cast<const float2*>(p.part_ml + (s * rows + row) * 2);
    if (ml.y != 0.0f) l += ml.y * at_exp2(ml.x - m);
  }
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;
  const int64_t tok = row / p.heads, h = row - tok * p.heads;
  T* out = static_cast<T*>(p.out) + tok * p.st[kPkO][0] + h * p.st[kPkO][1];
  for (int ch = 4 * lane; ch < p.dim; ch += 64) {
    at_f4 a = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int s = 0; s < p.splits; ++s) {
      const float2 ml = *reinterpret_cast<const float2*>(p.part_ml + (s * rows + row) * 2);
      if (ml.y != 0.0f) a += *reinterpret_cast<const at_f4*>(p.part_o + (s * rows + row) * p.dim + ch) * at_exp2(ml.x - m);
    }
    a *= inv;
    if constexpr (sizeof(T) == 2) {
      typedef __bf16 bf4 __attribute__((ext_vector_type(4)));
      *reinterpret_cast<uint2*>(reinterpret_cast<uint16_t*>(out) + ch) = __builtin_bit_cast(uint2, __builtin_convertvector(a, bf4));
    } else {
      *reinterpret_cast<at_f4*>(out + ch) = a;
    }
  }
  if (p.stats != nullptr && lane == 0)
    *reinterpret_cast<float2*>(p.stats + 4 * row) = pk_stats(m, l);
}

// dq, and delta into the statistics for the key side (alone when gq is null).
template <typename T, int DT>
__global__ void __launch_bounds__(256, sizeof(T) == 2 ? 2 : 1) pk_bwd_q_kernel(const PackParams p) {
  using Tile = PkTile<T, DT>;
  __shared__ __align__(16) unsigned char K0[Tile::BYTES], V0[Tile::BYTES], K1[Tile::BYTES], V1[Tile::BYTES];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, grp = lane >> 5, col = lane & 31;
  const PkQueries w(p, lane);
  if (w.r0 >= w.rows) return;
  const int r1 = min(w.r0 + kPkTile, w.rows);
  T* gq = static_cast<T*>(p.gq);
  if (w.w.seq < 0) {
    if (gq != nullptr) pk_zero_rows<T, 256>(w.r0, r1, p.dim, [&](int r) { return w.row(p, gq, kPkGQ, r); });
    return;
  }
  const int wr0 = w.r0 + 32 * wave, ri = wr0 + col, rc = min(ri, w.rows - 1);
  const bool valid = ri < w.rows;
  const int lim = valid ? w.seen(p, ri) : 0;
  const int end = w.seen(p, r1 - 1);
  const int wend = wr0 < w.rows ? w.seen(p, min(wr0 + 31, w.rows - 1)) : 0;
  const int wfull = wr0 + 31 < w.rows ? w.seen(p, wr0) : 0;
  const int chunks = (end + kPkChunk - 1) / kPkChunk;
  PkRow<T, DT> q, go;
  q.load(w.row(p, static_cast<const T*>(p.q), kPkQ, rc), valid, p.dim, grp);
  go.load(w.row(p, static_cast<const T*>(p.go), kPkGO, rc), valid, p.dim, grp);
  float m, ll, delta;
  {
    PkRow<T, DT> o;
    o.load(w.row(p, static_cast<const T*>(p.o), kPkO, rc), valid, p.dim, grp);
    delta = at_sum_halves(go.dot(o));
    float* st = p.stats + 4 * w.stat(p, rc);
    m = st[0];
    ll = st[1];
    if (valid && grp == 0) st[2] = delta;
  }
  if (gq == nullptr) return;
  const T* kp = static_cast<const T*>(p.k) + w.k_first * p.st[kPkK][0] + w.kv_head * p.st[kPkK][1];
  const T* vp = static_cast<const T*>(p.v) + w.k_first * p.st[kPkV][0] + w.kv_head * p.st[kPkV][1];
  at_f16 dq[DT / 32];
#pragma unroll
  for (int nd = 0; nd < DT / 32; ++nd) dq[nd] = at_zero16();

  auto stage = [&](unsigned char* K, unsigned char* V, int c) {
    PkStream<T, DT>::load(K, kp, p.st[kPkK][0], c * kPkChunk, w.m, p.dim);
    PkStream<T, DT>::load(V, vp, p.st[kPkV][0], c * kPkChunk, w.m, p.dim);
  };
  auto chunk = [&](const unsigned char* Kb, const unsigned char* Vb, int c) {
    const T* K = reinterpret_cast<const T*>(Kb);
    const T* V = reinterpret_cast<const T*>(Vb);
    const int k0 = c * kPkChunk;
    if (k0 >= wend) return;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      at_f16 s = pk_scores<T, DT>(K, 32 * h, q, col, grp), dp = pk_scores<T, DT>(V, 32 * h, go, col, grp);
      const bool full = k0 + 32 * h + 32 <= wfull;
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const float w2 = at_exp2(fmaf(s[i], p.scale2, -m) - ll) * (dp[i] - delta);
        s[i] = full || k0 + 32 * h + 8 * (i >> 2) + 4 * grp + (i & 3) < lim ? w2 : 0.0f;
      }
      pk_accumulate<T, DT>(dq, K, 32 * h, s, lane);
    }
  };
  if (chunks > 0) stage(K0, V0, 0);
  for (int c = 0; c < chunks; c += 2) {
    wait_vmem();
    __syncthreads();
    if (c + 1 < chunks) stage(K1, V1, c + 1);
    chunk(K0, V0, c);
    if (c + 1 >= chunks) break;
    wait_vmem();
    __syncthreads();
    if (c + 2 < chunks) stage(K0, V0, c + 2);
    chunk(K1, V1, c + 1);
  }
  __syncthreads();
  T* scratch = reinterpret_cast<T*>(wave == 0 ? K0 : wave == 1 ? V0 : wave == 2 ? K1 : V1);
  pk_store<T, DT>(dq, p.scale, scratch, p.dim, lane,
                  [&](int r) { return wr0 + r < w.rows ? w.row(p, gq, kPkGQ, wr0 + r) : static_cast<T*>(nullptr); });
}

// ---- keys on their own side: dk and dv ---------------------------------------------------------
// A workgroup takes 128 keys, 32 a wave in registers, and walks over the rows (tokens and heads of the key
// head's group) that see them, 64 at a time.
template <typename T, int DT>
__global__ void __launch_bounds__(256, sizeof(T) == 2 && DT <= 64 ? 2 : 1) pk_bwd_kv_kernel(const PackParams p) {
  using Tile = PkTile<T, DT>;
  __shared__ __align__(16) unsigned char Q0[Tile::BYTES], G0[Tile::BYTES], Q1[Tile::BYTES], G1[Tile::BYTES];
  __shared__ __align__(16) float row_m[2][kPkChunk], row_l[2][kPkChunk], row_d[2][kPkChunk];
  __shared__ __align__(16) int row_lim[2][kPkChunk];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, grp = lane >> 5, col = lane & 31;
  const int rest = static_cast<int>(blockIdx.x) / p.kv_heads, kv_head = static_cast<int>(blockIdx.x) - rest * p.kv_heads;
  // the first tiles, which the most queries of a causal sequence see, first
  const PkPlace w = pk_place<kPkTile>(p.k_offsets, p.sequences, p.k_rows, 1, rest, lane);
  const int b0 = w.tile * kPkTile;
  if (b0 >= w.own) return;
  const int b1 = min(b0 + kPkTile, w.own);
  T* gk = static_cast<T*>(p.gk);
  T* gv = static_cast<T*>(p.gv);
  auto key_row = [&](T* base, int t, int j) { return base + (static_cast<int64_t>(w.first) + j) * p.st[t][0] + kv_head * p.st[t][1]; };
  int m = 0, n = 0, q_first = 0;
  if (w.seq >= 0) {
    m = p.k_lengths != nullptr ? min(max(p.k_lengths[w.seq], 0), w.own) : w.own;
    q_first = min(max(p.q_offsets[w.seq], 0), p.q_rows);
    n = min(max(p.q_offsets[w.seq + 1], q_first), p.q_rows) - q_first;
  }
  if (b0 >= m || n == 0) {
    if (gk != nullptr) pk_zero_rows<T, 256>(b0, b1, p.dim, [&](int j) { return key_row(gk, kPkGK, j); });
    if (gv != nullptr) pk_zero_rows<T, 256>(b0, b1, p.dim, [&](int j) { return key_row(gv, kPkGV, j); });
    return;
  }
  const int rows = n * p.group, shift = m - n;
  const int wb0 = b0 + 32 * wave, kj = wb0 + col;
  const bool valid = kj < m;
  PkRow<T, DT> k, v;
  k.load(key_row(const_cast<T*>(static_cast<const T*>(p.k)), kPkK, min(kj, m - 1)), valid, p.dim, grp);
  v.load(key_row(const_cast<T*>(static_cast<const T*>(p.v)), kPkV, min(kj, m - 1)), valid, p.dim, grp);
  const T* qp = static_cast<const T*>(p.q) + q_first * p.st[kPkQ][0] + static_cast<int64_t>(kv_head) * p.group * p.st[kPkQ][1];
  const T* gp = static_cast<const T*>(p.go) + q_first * p.st[kPkGO][0] + static_cast<int64_t>(kv_head) * p.group * p.st[kPkGO][1];
  const float* sp = p.stats + 4 * (static_cast<int64_t>(q_first) * p.heads + kv_head * p.group);
  const int first = p.causal ? min(max(b0 - shift, 0), n) * p.group : 0;  // the first row that sees a key of the tile
  const int chunks = first < rows ? (rows - first + kPkChunk - 1) / kPkChunk : 0;
  at_f16 dk[DT / 32], dv[DT / 32];
#pragma unroll
  for (int nd = 0; nd < DT / 32; ++nd) dk[nd] = dv[nd] = at_zero16();

  float4 st;  // statistics of row threadIdx.x of the next tile
  int st_lim;
  auto stage = [&](unsigned char* Q, unsigned char* G, int c) {
    const int r0 = first + c * kPkChunk;
    PkStream<T, DT>::load_rows(Q, qp, p.st[kPkQ][0], p.st[kPkQ][1], p.group, r0, rows, p.dim);
    PkStream<T, DT>::load_rows(G, gp, p.st[kPkGO][0], p.st[kPkGO][1], p.group, r0, rows, p.dim);
  };
  auto load_stats = [&](int c) {
    const int r = first + c * kPkChunk + static_cast<int>(threadIdx.x);
    st = float4{0.0f, INFINITY, 0.0f, 0.0f};
    st_lim = 0;
    if (threadIdx.x < kPkChunk && r < rows) {
      const int t = r / p.group, g = r - t * p.group;
      st = *reinterpret_cast<const float4*>(sp + 4 * (static_cast<int64_t>(t) * p.heads + g));
      st_lim = p.causal ? min(max(t + shift + 1, 0), m) : m;
    }
  };
  auto store_stats = [&](int buf) {
    if (threadIdx.x < kPkChunk) {
      row_m[buf][threadIdx.x] = st.x;
      row_l[buf][threadIdx.x] = st.y;
      row_d[buf][threadIdx.x] = st.z;
      row_lim[buf][threadIdx.x] = st_lim;
    }
  };
  auto chunk = [&](const unsigned char* Qb, const unsigned char* Gb, int buf, int c) {
    const T* Q = reinterpret_cast<const T*>(Qb);
    const T* G = reinterpret_cast<const T*>(Gb);
    const int r0 = first + c * kPkChunk;
    if (wb0 >= m || (p.causal && (min(r0 + kPkChunk, rows) - 1) / p.group + shift < wb0)) return;
    // every row sees every key of the wave
    const bool full = r0 + kPkChunk <= rows && (p.causal ? r0 / p.group + shift >= wb0 + 31 && wb0 + 32 <= m : wb0 + 32 <= m);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      at_f16 s = pk_scores<T, DT>(Q, 32 * h, k, col, grp), dp = pk_scores<T, DT>(G, 32 * h, v, col, grp);
#pragma unroll
      for (int c4 = 0; c4 < 4; ++c4) {
        const int at = 32 * h + 8 * c4 + 4 * grp;
        const at_f4 mm = *reinterpret_cast<const at_f4*>(&row_m[buf][at]), ll = *reinterpret_cast<const at_f4*>(&row_l[buf][at]);
        const at_f4 dd = *reinterpret_cast<const at_f4*>(&row_d[buf][at]);
        const int4 lm = *reinterpret_cast<const int4*>(&row_lim[buf][at]);
        const int lim[4] = {lm.x, lm.y, lm.z, lm.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int i = 4 * c4 + j;
          const bool sees = full || kj < lim[j];
          s[i] = sees ? at_exp2(fmaf(s[i], p.scale2, -mm[j]) - ll[j]) : 0.0f;
          dp[i] = sees ? s[i] * (dp[i] - dd[j]) : 0.0f;
        }
      }
      pk_accumulate<T, DT>(dv, G, 32 * h, s, lane);
      pk_accumulate<T, DT>(dk, Q, 32 * h, dp, lane);
    }
  };
  if (chunks > 0) {
    load_stats(0);
    stage(Q0, G0, 0);
  }
  for (int c = 0; c < chunks; c += 2) {
    store_stats(0);
    wait_vmem();
    __syncthreads();
    if (c + 1 < chunks) {
      load_stats(c + 1);
      stage(Q1, G1, c + 1);
    }
    chunk(Q0, G0, 0, c);
    if (c + 1 >= chunks) break;
    store_stats(1);
    wait_vmem();
    __syncthreads();
    if (c + 2 < chunks) {
      load_stats(c + 2);
      stage(Q0, G0, c + 2);
    }
    chunk(Q1, G1, 1, c + 1);
  }
  __syncthreads();
  T* scratch = reinterpret_cast<T*>(wave == 0 ? Q0 : wave == 1 ? G0 : wave == 2 ? Q1 : G1);
  // keys from m on (rows of the range behind the sequence's keys) hold zeros: their scores never counted
  if (gk != nullptr)
    pk_store<T, DT>(dk, p.scale, scratch, p.dim, lane, [&](int r) { return wb0 + r < b1 ? key_row(gk, kPkGK, wb0 + r) : static_cast<T*>(nullptr); });
  if (gv != nullptr)
    pk_store<T, DT>(dv, 1.0f, scratch, p.dim, lane, [&](int r) { return wb0 + r < b1 ? key_row(gv, kPkGV, wb0 + r) : static_cast<T*>(nullptr); });
}

}  // namespace msda
