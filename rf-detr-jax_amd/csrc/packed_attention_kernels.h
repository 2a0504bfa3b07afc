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
// Finding the tile. The segments (the rows before the first sequence, the sequences, the rows behind the
// last) of some rows have at most rows / 128 + segments tiles of 128 rows, so the grid is known without the
// lengths, and a workgroup finds its tile by adding up the segments' tiles (pk_place): no length is read back
// by the host and no launch prepares a table. Offsets are clamped to the tensors' rows: wrong ones give
// wrong values and no access out of bounds. Rows outside every sequence are written as zeros.
//
// Layouts of the products as in attention_kernels.h: scores are formed transposed (streamed rows x own
// rows), a lane owns one own row (its softmax statistics stay in the lane), and the weights in their
// result registers are the B operand of the next product, whose A operand is read from the streamed
// tile by transposing LDS reads. Streamed tiles of 64 rows lie in LDS as swizzled rows, written by
// buffer loads into LDS (no registers, two buffers, one barrier a tile), which bring zeros for rows past a
// sequence's end and channels past head_dim.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>
#include <type_traits>
#include <utility>

#include "attention_common.h"
#include "msda_kernels.h"  // bf16_t, wait_vmem
#include "packed_attention_parts.h"

namespace msda {

enum PackTensor { kPkQ = 0, kPkK, kPkV, kPkO, kPkGO, kPkGQ, kPkGK, kPkGV, kPkTensors };

struct PackParams {
  const void* q;
  const void* k;
  const void* v;
  const void* o;   // backward: the forward output
  const void* go;  // backward: grad of the output
  void* out;
  void* rest;  // forward: what out's rounding left (out's type and strides), or null; backward: the same, read
  void* gq;  // backward outputs (each may be null)
  void* gk;
  void* gv;
  float* stats;    // [q_rows * heads][4]: m, log2 l (forward; the backward reads them); row (token, head)
  float* numbers;  // backward: the same and two numbers more (pk_bwd_q_kernel), for the key side; stats itself, or a
                   // buffer of the call; null when neither gk nor gv is wanted
  const int32_t* q_offsets;  // [sequences + 1]
  const int32_t* k_offsets;  // [sequences + 1]
  const int32_t* k_lengths;  // [sequences], or null: all rows of a sequence's range
  float* part_o;             // split forward: [splits][q_rows * heads][dim], sums relative to part_ml's m
  float* part_ml;            // [splits][q_rows * heads][2]: m, l
  int32_t* part_n;           // [q_rows * heads]: the row's parts
  float* part_kv;            // key side: [splits][dk, dv][k_rows * kv_heads][dim]
  int64_t st[kPkTensors][2];  // element strides (row, head) of each tensor
  int sequences, q_rows, k_rows, heads, kv_heads, group, dim, causal;
  int splits;    // at most so many workgroups share a tile's streamed rows
  int part;      // forward: chunks of one of them, unless that makes more
  int slots;     // tiles of the kernel's own side
  float scale;   // of the scores
  float scale2;  // scale log2(e)
};

constexpr int kPkPart = 32;  // chunks of a workgroup on the key side, unless that makes more parts than the host gave room for
constexpr int kPkJoin = 32;   // workgroups that join a key tile's parts

__device__ __align__(16) const uint32_t pk_zeros[4] = {0u, 0u, 0u, 0u};

// ---- the workgroup's place ---------------------------------------------------------------------

// First row of segment s, 0 <= s <= sequences + 2, clamped to the tensor (a load without a branch, so that several
// are under way together).
__device__ __forceinline__ int pk_bound(const int32_t* offsets, int s, int sequences, int rows) {
  const int x = min(max(offsets[min(max(s - 1, 0), sequences)], 0), rows);
  return s == 0 ? 0 : s >= sequences + 2 ? rows : x;
}

struct PkPlace {
  int seq;         // the sequence, or -1: rows outside every sequence
  int first;       // first row of the segment in the own tensor
  int own;         // its rows (tokens)
  int tile;        // tile of the segment
};

// Sum over the lanes up to this one.
__device__ __forceinline__ int pk_scan(int x) {
  x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xf, 0xf, true);  // within rows of 16 lanes
  x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xf, 0xf, true);
  x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xf, 0xf, true);
  x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xf, 0xf, true);
  x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xa, 0xf, false);  // lane 15's to the next row
  x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xc, 0xf, false);  // lane 31's to the upper half
  return x;
}

constexpr int kPkCounted = 1024;  // segments whose tiles a wave counts

// Tile, or unit of a tile's work, of workgroup `index` of a grid. LAST_FIRST: a segment's last one first. `unit`: rows of
// a tile's matrix to a row of the tensor; `alike`: units are of about one size, so no order is better. No rows
// (own = 0) for the grid's tiles that do not exist.
// Up to kPkCounted segments the wave adds up all segments' units, count(s, rows) of segment s, and w.tile is the
// unit's number in its segment. So the units that do not exist are the grid's last. That matters: the hardware
// hands workgroups to its shader engines in turn whether they end at once or not, and with empty ones among
// them (sequences of 128 rows: every second one) half of the CUs stood idle: forward of 128 times 128 queries over
// 1,024 keys, 8 heads, 173 us for 140 in bf16 at 128 channels, 540 for 287 in f32 at 64. The counting has its price,
// the loads of 2 segments / 64 offsets a lane, one behind the other, and the sorting of up to 64 segments another: 128
// tokens each that see themselves, 8 heads, bf16 at 64 channels, 62 sequences 17.7 us, 63 10.0, 1,022 267, and 1,023,
// searched, 96.
// Of more segments it searches, 64 at a time, among `slots` tiles, with segment s at tile floor(first row / 128) + s,
// behind which it has room for ceil(rows / 128).
template <bool LAST_FIRST, typename Count>
__device__ __forceinline__ PkPlace pk_place(const int32_t* offsets, int sequences, int rows, int unit, int index, int slots, int lane, bool alike,
                                            Count&& count) {
  const int segments = sequences + 2;
  PkPlace w{-1, 0, 0, 0};
  int s;
  if (segments <= kPkCounted) {
    const int per = (segments + 63) / 64;
    auto units = [&](int s) {
      const int n = pk_bound(offsets, s + 1, sequences, rows) - pk_bound(offsets, s, sequences, rows), units = count(s, max(n, 1));
      return s >= segments || n <= 0 ? 0 : units;
    };
    if (per == 1 && !alike) {  // the longest segment first: the work of its tiles sets the time if they start last
      const int mine = units(lane), length = lane >= segments ? 0 : pk_bound(offsets, lane + 1, sequences, rows) - pk_bound(offsets, lane, sequences, rows);
      int base = 0;
      for (int j = 0; j < segments; ++j) {
        const int other = __builtin_amdgcn_readlane(length, j), more = __builtin_amdgcn_readlane(mine, j);
        base += other > length || (other == length && j < lane) ? more : 0;
      }
      const uint64_t here = __ballot(base <= index && index < base + mine);
      if (here == 0) return w;
      s = static_cast<int>(__builtin_ctzll(here));
      w.tile = index - __builtin_amdgcn_readlane(base, s);
      if (LAST_FIRST) w.tile = __builtin_amdgcn_readlane(mine, s) - 1 - w.tile;
    } else {
      int mine = 0;
      for (int i = 0; i < per; ++i) mine += units(lane * per + i);
      int end = pk_scan(mine);
      const int total = __builtin_amdgcn_readlane(end, 63), t = LAST_FIRST ? total - 1 - index : index;
      if (t < 0 || t >= total) return w;
      int at = static_cast<int>(__popcll(__ballot(end <= t))), base = __builtin_amdgcn_readlane(end - mine, at);
      s = at * per;
      if (per > 1) {
        mine = lane < per ? units(s + lane) : 0;
        end = base + pk_scan(mine);
        at = static_cast<int>(__popcll(__ballot(end <= t)));
        base = __builtin_amdgcn_readlane(end - mine, at);
        s += at;
      }
      w.tile = t - base;
      // Offsets that rise have fewer units than the grid. Of ones that fall and rise again the sum may pass 32 bits.
      if (at > 63 || static_cast<uint32_t>(w.tile) >= static_cast<uint32_t>(__builtin_amdgcn_readlane(mine, at & 63))) return PkPlace{-1, 0, 0, 0};
    }
  } else {
    const int slot = LAST_FIRST ? slots - 1 - index : index;
    int lo = 0, hi = segments;
    auto at = [&](int s) { return static_cast<int>(static_cast<uint32_t>(pk_bound(offsets, s, sequences, rows)) * unit / kPkTile) + s; };
    while (hi - lo > 1) {
      const int step = (hi - lo + 63) / 64, x = lo + lane * step;
      const int n = max(1, static_cast<int>(__popcll(__ballot(x < hi && at(x) <= slot))));
      lo += (n - 1) * step;
      hi = min(hi, lo + step);
    }
    s = __builtin_amdgcn_readfirstlane(lo);
    w.tile = slot - at(s);
    if (w.tile < 0) return PkPlace{-1, 0, 0, 0};  // only where the offsets fall
  }
  w.first = pk_bound(offsets, s, sequences, rows);
  w.own = max(0, pk_bound(offsets, s + 1, sequences, rows) - w.first);
  w.seq = s >= 1 && s <= sequences ? s - 1 : -1;
  return w;
}

// The place in line of number `index` of `count`: every second round is walked backwards. Workgroups go to the 8
// XCDs, and there to 4 shader engines, in turn, R tiles to a round; a causal sequence's tiles fall by size, and
// walked in one direction the first of them would get the largest of every round.
__device__ __forceinline__ int pk_line(int index, int count, int kv_heads) {
  const int shift = 5 - min(5, static_cast<int>(__builtin_ctz(kv_heads))), round = index >> shift;
  if ((round & 1) == 0 || (round + 1) << shift > count) return index;
  return (2 * round + 1 << shift) - 1 - index;
}

__device__ __forceinline__ int pk_tiles(int rows, int unit) { return static_cast<int>((static_cast<uint32_t>(rows) * unit + (kPkTile - 1)) / kPkTile); }

// The keys of sequence `seq`: first row and number.
struct PkRange {
  int first, count;
  __device__ __forceinline__ PkRange(const PackParams& p, int seq) {
    first = min(max(p.k_offsets[seq], 0), p.k_rows);
    const int end = min(max(p.k_offsets[seq + 1], first), p.k_rows);
    count = p.k_lengths != nullptr ? min(max(p.k_lengths[seq], 0), end - first) : end - first;
  }
};

// ---- operands ----------------------------------------------------------------------------------

using PkLds = const MSDA_LDS unsigned char*;

// DT: channels that the products run over (head_dim rounded up to 32); a tile's rows lie DP apart.
template <typename T, int DT>
struct PkTile {
  static constexpr int DP = DT == 96 ? 128 : DT;
  static constexpr int E = 16 / static_cast<int>(sizeof(T));  // elements of a 16-byte chunk
  static constexpr int CPR = DP / E;                          // chunks of a row
  static constexpr int ROW = DP * static_cast<int>(sizeof(T));  // bytes of a row
  static constexpr int BYTES = kPkChunk * ROW;
  // 16-byte chunk c of row r sits at slot c ^ swizzle(r), so that what one read takes together falls on
  // distinct banks (256 bytes a clock): 16 rows of one chunk (operands along the channels); 4 rows of 4
  // chunks (bf16, transposing reads: rows that share a 256-byte line differ in the slot's upper bits); 8
  // chunks of rows 4 apart (f32, along the rows: their halves of a line differ). With r % 16 for a swizzle
  // the transposing reads met 4 rows on the same banks, and the forward at 128 channels spent 60 % of its
  // LDS time on conflicts.
  static __device__ __forceinline__ constexpr int swizzle(int r) {
    if (sizeof(T) == 2) {
      if (CPR == 16) return ((r & 3) << 2) | ((r >> 2) & 3);
      if (CPR == 8) return (((r >> 1) & 1) << 2) | ((r >> 2) & 3);
      return (r >> 2) & 3;
    }
    return CPR >= 16 ? ((((r >> 2) & 1) << 3) | (((r >> 3) & 1) << 2) | (r & 3)) : ((r >> 1) & 7);
  }
};

// A lane's byte offsets in a tile. The chunks that one lane reads differ in bits that neither its row's
// swizzle nor a carry reaches, so they are an exclusive or with a constant away from one offset, and rows
// 8 apart the mask kRows8: an offset costs one instruction, and a few registers serve a whole tile.
template <typename T, int DT>
struct PkLane {
  using Tile = PkTile<T, DT>;
  static constexpr uint32_t kRows8 = 32;  // bf16: swizzle(r) ^ swizzle(r + 8), as bytes
  uint32_t row;  // row col, chunk grp: operands along the channels
  uint32_t tr;   // bf16: rows 4 grp + (lane % 16) / 4, channels 16 (lane / 16 % 2) + 4 (lane % 4)
                 // f32: row 4 grp, channel col: operands along the rows
  __device__ __forceinline__ explicit PkLane(int lane) {
    const int grp = lane >> 5, col = lane & 31;
    row = col * Tile::ROW + ((grp ^ Tile::swizzle(col)) << 4);
    if constexpr (sizeof(T) == 2) {
      const int g = (lane >> 4) & 1, r = lane & 15, ro = 4 * grp + (r >> 2);
      tr = ro * Tile::ROW + (((2 * g + ((r & 3) >> 1)) ^ Tile::swizzle(ro)) << 4) + (r & 1) * 8;
    } else {
      tr = 4 * grp * Tile::ROW + (((col >> 2) ^ Tile::swizzle(4 * grp)) << 4) + (col & 3) * 4;
    }
  }
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

__device__ __forceinline__ uint2 pk_read_tr(PkLds p) {
  return __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((MSDA_LDS at_s4*)(p)));
}

// f(0) .. f(N - 1) with the number as a constant.
template <int I>
using PkInt = std::integral_constant<int, I>;
template <typename F, int... I>
__device__ __forceinline__ void pk_for_each(F&& f, std::integer_sequence<int, I...>) {
  (f(PkInt<I>{}), ...);
}
template <int N, typename F>
__device__ __forceinline__ void pk_for(F&& f) {
  pk_for_each(f, std::make_integer_sequence<int, N>{});
}

// N products, the operand of each read from LDS PF products ahead. The barriers hold everything in the order
// that it is written in (MAY: but the kinds of instructions that may pass), the vector work `beside` a product
// included: left to itself the compiler reads an operand, waits for it, and multiplies, one at a time, and all
// vector work after that.
template <int N, int PF, int MAY = 0, typename Read, typename Use, typename Beside>
__device__ __forceinline__ void pk_pipe(Read&& read, Use&& use, Beside&& beside) {
  decltype(read(PkInt<0>{})) a[PF];
  pk_for<PF>([&](auto i) { a[i] = read(i); });
  __builtin_amdgcn_sched_barrier(MAY);
  pk_for<N>([&](auto i) {
    use(i, a[i % PF]);
    if constexpr (i + PF < N) a[i % PF] = read(PkInt<i + PF>{});
    beside(i);
    __builtin_amdgcn_sched_barrier(MAY);
  });
}

// Vector work beside the KS products of a phase: a product's result is there one product later, so step t
// takes part t - 1 of KS - 1 of the 16 registers.
template <int KS, int T, typename F>
__device__ __forceinline__ void pk_beside(F&& f) {
  if constexpr (T >= 1) {
    constexpr int lo = 16 * (T - 1) / (KS - 1), hi = 16 * T / (KS - 1);
    pk_for<hi - lo>([&](auto i) { f(lo + i); });
  }
}

// Operands of one 32-row block of a tile. Scores of block X against the lane's row r: register i of the
// result holds streamed row 8 (i / 4) + 4 grp + i % 4. Sums X^T w, w in result-layout registers: register
// i of acc[nd] holds channel 32 nd + 8 (i / 4) + 4 grp + i % 4 of the lane's row; bf16: w is rounded to
// bf16 for the product (half a step, 2^-8 of each weight at most: as much as the inputs' and the result's
// own rounding).
template <typename T, int DT>
struct PkProducts;

template <int DT>
struct PkProducts<bf16_t, DT> {
  using T = bf16_t;
  static constexpr int ROW = PkTile<T, DT>::ROW, KS = DT / 16, ND = DT / 32;
  static constexpr int kScores = KS, kSums = 2 * ND;  // products of a block
  static __device__ __forceinline__ at_bf8 row_operand(PkLds X, const PkLane<T, DT>& at, int i) {
    return *reinterpret_cast<const MSDA_LDS at_bf8*>(X + (at.row ^ (i << 5)));
  }
  static __device__ __forceinline__ void score(at_f16& s, const at_bf8& a, const at_bf8& b) {
    s = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, s, 0, 0, 0);
  }
  static __device__ __forceinline__ void score(at_f16& s, const at_bf8& a, const PkRow<T, DT>& r, int i) { score(s, a, r.x[i]); }
  // product j: rows 16 (j / ND) .. + 15, channels of block j % ND
  static __device__ __forceinline__ at_bf8 sum_operand(PkLds X, const PkLane<T, DT>& at, int j) {
    const int s = j / ND, nd = j % ND;
    const uint32_t o = at.tr ^ (nd << 6);
    return at_bf8_of(pk_read_tr(X + o + 16 * s * ROW), pk_read_tr(X + (o ^ PkLane<T, DT>::kRows8) + (16 * s + 8) * ROW));
  }
  struct Weights {
    at_bf8 b[2];
    __device__ __forceinline__ void set(const at_f16& w) {
      b[0] = at_bf8_regs(w, 0);
      b[1] = at_bf8_regs(w, 8);
    }
  };
  static __device__ __forceinline__ void sum(at_f16 (&acc)[ND], const at_bf8& a, const Weights& w, int j) {
    acc[j % ND] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, w.b[j / ND], acc[j % ND], 0, 0, 0);
  }
};

template <int DT>
struct PkProducts<float, DT> {
  using T = float;
  static constexpr int ROW = PkTile<T, DT>::ROW, ND = DT / 32;
  static constexpr int kScores = DT / 8, kSums = 16;  // steps of a block (4 and ND products each)
  static __device__ __forceinline__ at_f4 row_operand(PkLds X, const PkLane<T, DT>& at, int c) {
    return *reinterpret_cast<const MSDA_LDS at_f4*>(X + (at.row ^ (c << 5)));
  }
  static __device__ __forceinline__ void score(at_f16& s, const at_f4& a, const PkRow<T, DT>& r, int c) {
#pragma unroll
    for (int j = 0; j < 4; ++j) s = __builtin_amdgcn_mfma_f32_32x32x2f32(a[j], r.x[c][j], s, 0, 0, 0);
  }
  struct Operand {
    float a[ND];
  };
  static __device__ __forceinline__ Operand sum_operand(PkLds X, const PkLane<T, DT>& at, int i) {
    const int ro = 8 * (i >> 2) + (i & 3);  // row 4 grp + ro: the swizzle's bits of 4 grp (in at.tr) and of ro do not meet
    const uint32_t x = PkTile<T, DT>::swizzle(ro);
    Operand o;
#pragma unroll
    for (int nd = 0; nd < ND; ++nd) o.a[nd] = *reinterpret_cast<const MSDA_LDS float*>(X + (at.tr ^ ((x ^ (8 * nd)) << 4)) + ro * ROW);
    return o;
  }
  struct Weights {
    at_f16 b;
    __device__ __forceinline__ void set(const at_f16& w) { b = w; }
  };
  static __device__ __forceinline__ void sum(at_f16 (&acc)[ND], const Operand& o, const Weights& w, int i) {
#pragma unroll
    for (int nd = 0; nd < ND; ++nd) acc[nd] = __builtin_amdgcn_mfma_f32_32x32x2f32(o.a[nd], w.b[i], acc[nd], 0, 0, 0);
  }
};

// s += scores of X with x, t += scores of Y with y.
template <typename T, int DT, int PF>
__device__ __forceinline__ void pk_scores2(at_f16& s, PkLds X, const PkRow<T, DT>& x, at_f16& t, PkLds Y, const PkRow<T, DT>& y,
                                           const PkLane<T, DT>& at) {
  using P = PkProducts<T, DT>;
  constexpr int N = P::kScores;
  pk_pipe<2 * N, PF, 0x6>([&](auto i) { return P::row_operand(i < N ? X : Y, at, i % N); },
                     [&](auto i, const auto& a) {
                       if constexpr (i < N) P::score(s, a, x, i);
                       else P::score(t, a, y, i - N);
                     },
                     [](auto) {});
}

// acc += X^T w
template <typename T, int DT, int PF>
__device__ __forceinline__ void pk_accumulate(at_f16 (&acc)[DT / 32], PkLds X, const at_f16& w, const PkLane<T, DT>& at) {
  using P = PkProducts<T, DT>;
  typename P::Weights b;
  b.set(w);
  pk_pipe<P::kSums, PF, 0x6>([&](auto i) { return P::sum_operand(X, at, i); }, [&](auto i, const auto& a) { P::sum(acc, a, b, i); }, [](auto) {});
}

// ax += X^T wx, ay += Y^T wy
template <typename T, int DT, int PF>
__device__ __forceinline__ void pk_accumulate2(at_f16 (&ax)[DT / 32], PkLds X, const at_f16& wx, at_f16 (&ay)[DT / 32], PkLds Y, const at_f16& wy,
                                               const PkLane<T, DT>& at) {
  using P = PkProducts<T, DT>;
  constexpr int N = P::kSums;
  typename P::Weights bx, by;
  bx.set(wx);
  by.set(wy);
  pk_pipe<2 * N, PF, 0x6>([&](auto i) { return P::sum_operand(i < N ? X : Y, at, i % N); },
                     [&](auto i, const auto& a) {
                       if constexpr (i < N) P::sum(ax, a, bx, i);
                       else P::sum(ay, a, by, i - N);
                     },
                     [](auto) {});
}

typedef __bf16 pk_bf16 __attribute__((ext_vector_type(16)));
typedef __bf16 pk_bf4 __attribute__((ext_vector_type(4)));

// What the rounding to bf16 leaves.
__device__ __forceinline__ at_f16 pk_rest(const at_f16& x) { return x - __builtin_convertvector(__builtin_convertvector(x, pk_bf16), at_f16); }

// A wave's LDS accesses are in order; this keeps the compiler from exchanging them.
__device__ __forceinline__ void pk_wave_sync() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// Writes acc * f (f: of the lane's row) as rows of T: through the wave's LDS scratch, half a tile of the same
// layout, so that each lane stores 16 bytes and the wave whole rows. `row(r)`: the address of own row r of the
// wave's 32, or null. REST: what the rounding to T leaves of them instead.
template <typename T, int DT, bool REST = false, typename R>
__device__ __forceinline__ void pk_store(const at_f16 (&acc)[DT / 32], float f, unsigned char* scratch, int dim, int lane, R&& row) {
  using Tile = PkTile<T, DT>;
  const int grp = lane >> 5, col = lane & 31;
  unsigned char* mine = scratch + col * Tile::ROW;
#pragma unroll
  for (int nd = 0; nd < DT / 32; ++nd) {
    at_f16 v = acc[nd] * f;
    if constexpr (REST) v = pk_rest(v);
#pragma unroll
    for (int c = 0; c < 4; ++c) {  // channels 32 nd + 8 c + 4 grp .. + 3
      const at_f4 x = {v[4 * c], v[4 * c + 1], v[4 * c + 2], v[4 * c + 3]};
      if constexpr (sizeof(T) == 2)
        *reinterpret_cast<uint2*>(mine + (((4 * nd + c) ^ Tile::swizzle(col)) << 4) + 8 * grp) = __builtin_bit_cast(uint2, __builtin_convertvector(x, pk_bf4));
      else
        *reinterpret_cast<at_f4*>(mine + (((8 * nd + 2 * c + grp) ^ Tile::swizzle(col)) << 4)) = x;
    }
  }
  pk_wave_sync();
  constexpr int C = DT / Tile::E;
#pragma unroll 2
  for (int k = 0; k < C / 2; ++k) {
    const int idx = lane + 64 * k, r = idx / C, c = idx - r * C;
    T* to = row(r);
    if (to != nullptr && c * Tile::E < dim)
      *reinterpret_cast<uint4*>(to + c * Tile::E) = *reinterpret_cast<const uint4*>(scratch + r * Tile::ROW + ((c ^ Tile::swizzle(r)) << 4));
  }
  pk_wave_sync();
}

// Rows of zeros: own rows [r0, r1) of the matrix, `row(r)` their addresses, by the whole workgroup.
template <typename T, typename R>
__device__ __forceinline__ void pk_zero_rows(int r0, int r1, int dim, R&& row) {
  constexpr int E = 16 / static_cast<int>(sizeof(T));
  const int c = dim / E;
  for (int idx = threadIdx.x; idx < (r1 - r0) * c; idx += 64 * kPkWaves) {
    const int r = idx / c;
    *reinterpret_cast<uint4*>(row(r0 + r) + E * (idx - r * c)) = uint4{0u, 0u, 0u, 0u};
  }
}

// ---- streaming ---------------------------------------------------------------------------------

constexpr int kPkFar = 0x7fffff00;  // a byte offset behind every tile: its transfer brings zeros

// A buffer of `bytes` from p on (both uniform): transfers from behind it bring zeros, so rows past a
// sequence's end and channels past head_dim need no test of their own. Buffer instructions also count as
// memory accesses alone; global ones into LDS count as LDS accesses too, after which every wait for an
// operand from LDS would wait for all of them.
__device__ __forceinline__ __amdgpu_buffer_rsrc_t pk_buffer(const void* p, int bytes) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(p), 0, bytes, 0x00020000);
}

// The workgroup's barrier, with the wave's transfers into LDS landed and its LDS reads done.
__device__ __forceinline__ void pk_barrier() {
  wait_vmem();
  __syncthreads();
}

// The transfers of one 64-row tile by the workgroup: piece u is row u / CPR, slot u % CPR,
// which holds the row's chunk slot ^ swizzle(row). A thread's pieces are kStep rows apart. Row strides are
// below 2^22 elements, a group's heads within 2^27 (the host's checks), so a tile's offsets fit 31 bits.
template <typename T, int DT>
struct PkStream {
  using Tile = PkTile<T, DT>;
  static constexpr int kStep = 64 * kPkWaves / Tile::CPR, NV = kPkChunk / kStep;
  static_assert(kStep * NV == kPkChunk, "whole pieces");
  static __device__ __forceinline__ void transfer(__amdgpu_buffer_rsrc_t src, int offset, unsigned char* lds, int v) {
    const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x >> 6));
    __builtin_amdgcn_raw_ptr_buffer_load_lds(src, (MSDA_LDS void*)(lds + 64 * (kPkWaves * v + wave) * 16), 16, offset, 0, 0, 0);
  }
  // row and channel of piece v of thread t
  static __device__ __forceinline__ int row(int t, int v) { return t / Tile::CPR + kStep * v; }
  static __device__ __forceinline__ int channel(int t, int v) { return Tile::E * ((t % Tile::CPR) ^ Tile::swizzle(row(t, v))); }
  // Rows [first, first + 64) of two tensors (row r at base + r stride), rows from `end` on as zeros (all of them
  // when there is no such tile), into two tiles: 2 NV pieces, which are issued one at a time between other
  // work. A piece keeps the CU's address unit busy for 16 clocks, and the waves that issue theirs together wait
  // for one another: together at the start of a chunk they took 480 of the forward's 3,300 clocks a chunk.
  struct Pair {
    __amdgpu_buffer_rsrc_t x, y;
    unsigned char* lx;
    unsigned char* ly;
    int sx, sy, dim;
    __device__ __forceinline__ Pair(unsigned char* to_x, const T* bx, int64_t stride_x, unsigned char* to_y, const T* by, int64_t stride_y, int first,
                                    int end, int d)
        : lx(to_x), ly(to_y), sx(static_cast<int>(stride_x * static_cast<int>(sizeof(T)))), sy(static_cast<int>(stride_y * static_cast<int>(sizeof(T)))), dim(d) {
      // (by hand: the compiler takes a clamp to the vector unit, and a buffer in vector registers to a loop)
      const int rows = __builtin_amdgcn_readfirstlane(min(max(end - first, 0), kPkChunk));
      x = pk_buffer(bx + first * stride_x, rows * sx);
      y = pk_buffer(by + first * stride_y, rows * sy);
    }
    template <int I>
    __device__ __forceinline__ void piece() const {
      constexpr int v = I % NV;
      const int t = static_cast<int>(threadIdx.x), ch = channel(t, v);
      const int o = dim == Tile::DP || ch < dim ? row(t, v) * (I < NV ? sx : sy) + ch * static_cast<int>(sizeof(T)) : kPkFar;
      transfer(I < NV ? x : y, o, I < NV ? lx : ly, v);
    }
    __device__ __forceinline__ void all() const {
      pk_for<2 * NV>([&](auto i) { piece<i>(); });
    }
  };
};

// A causal chunk that not every row of the workgroup sees whole: the weights of its unseen pairs are zeros, and
// zero times an infinity or NaN of an unseen row would reach the sums. So such a tile is searched first (one
// round of 16-byte reads and a barrier, for the chunks on the diagonal alone), values that are no finite numbers
// become zeros, and the rows that held some are marked in `bad`, for those who see them.
typedef uint16_t pk_u2 __attribute__((ext_vector_type(2)));
template <typename T, int DT>
__device__ __forceinline__ void pk_settle(unsigned char* tile, uint32_t* bad) {
  using Tile = PkTile<T, DT>;
  constexpr bool bf = sizeof(T) == 2;
  constexpr int N = Tile::BYTES / (16 * 64 * kPkWaves);
  int thread = threadIdx.x;
  asm volatile("" : "+v"(thread));  // addresses formed here, not kept in registers from before the loop
  uint4* mine = reinterpret_cast<uint4*>(tile) + thread;
  // the largest magnitude, as an integer: of the upper and of the lower halves in bf16
  uint32_t most = 0;
  auto larger = [](uint32_t a, uint32_t b) {
    if constexpr (bf) return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(pk_u2, a), __builtin_bit_cast(pk_u2, b)));
    else return max(a, b);
  };
  constexpr uint32_t kMagnitude = bf ? 0x7fff7fffu : 0x7fffffffu;
#pragma unroll 1  // (unrolled, the key side's kernel spills at 128 channels: 277 us for 264 over 8,848 tokens of 16 heads)
  for (int v = 0; v < N; ++v) {
    const uint4 x = mine[64 * kPkWaves * v];
    most = larger(larger(larger(most, x.x & kMagnitude), larger(x.y & kMagnitude, x.z & kMagnitude)), x.w & kMagnitude);
  }
  if (most < 0x7f800000u && (!bf || (most & 0xffffu) < 0x7f80u)) return;
#pragma unroll 1
  for (int v = 0; v < N; ++v) {
    const int r = (thread + 64 * kPkWaves * v) / Tile::CPR;
    auto settled = [](uint32_t w) {
      if ((w & 0x7f800000u) == 0x7f800000u) w &= bf ? 0xffffu : 0u;
      if (bf && (w & 0x7f80u) == 0x7f80u) w &= 0xffff0000u;
      return w;
    };
    const uint4 x = mine[64 * kPkWaves * v], y = {settled(x.x), settled(x.y), settled(x.z), settled(x.w)};
    if (x.x == y.x && x.y == y.y && x.z == y.z && x.w == y.w) continue;
    mine[64 * kPkWaves * v] = y;
    atomicOr(bad + (r >> 5), 1u << (r & 31));
  }
}
__device__ __forceinline__ uint64_t pk_settled(const uint32_t* bad) {
  __syncthreads();
  return static_cast<uint64_t>(static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(static_cast<int>(bad[1])))) << 32 |
         static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(static_cast<int>(bad[0])));
}

// The rows r = t G + g of a key head's queries (G <= 64), in chunks of whole tokens, at most 64 rows: a row's
// place in its chunk gives its token and head whatever the chunk.
struct PkRows {
  int group, tokens;  // tokens of a chunk
  uint32_t magic;     // x / group = x magic >> 16 for x < 64: x (magic group - 2^16) < 2^16
  __device__ __forceinline__ explicit PkRows(int g) : group(g), tokens(kPkChunk / g), magic((65536 + g - 1) / g) {}
  __device__ __forceinline__ int token(int x) const { return static_cast<int>((static_cast<uint32_t>(x) * magic) >> 16); }
};

// ---- queries on their own side: forward and dq -------------------------------------------------

struct PkQueries {
  PkPlace w;
  int kv_head;      // key head
  int split, parts; // the workgroup's part of the tile's keys, of so many (forward)
  int rows, r0;     // rows of the sequence's matrix, first of the workgroup's; none: no work
  int64_t k_first;  // first key row
  int m, shift;     // keys; a row of token t sees the keys below min(m, t + shift + 1)
  template <bool SPLIT>
  __device__ PkQueries(const PackParams& p, int lane, std::bool_constant<SPLIT>) {
    // key heads fastest: with 8 of them each stays on one XCD, whose L2 then holds its keys; the last
    // tiles, which see the most keys of a causal sequence, first
    const int b = static_cast<int>(blockIdx.x), rest = b / p.kv_heads;
    kv_head = b - rest * p.kv_heads;
    parts = 1;
    split = 0;
    const bool counted = p.sequences + 2 <= kPkCounted, shared = SPLIT && p.splits > 1;
    if (!shared) {
      w = pk_place<true>(p.q_offsets, p.sequences, p.q_rows, p.group, pk_line(rest, p.slots, p.kv_heads), p.slots, lane, false, [&](int, int n) { return pk_tiles(n, p.group); });
    } else {
      split = counted ? 0 : rest / p.slots;
      const int line = pk_line(rest - split * p.slots, counted ? p.slots * p.splits : p.slots, p.kv_heads);
      w = pk_place<true>(p.q_offsets, p.sequences, p.q_rows, p.group, line, p.slots, lane, true, [&](int s, int n) {
        const int tiles = pk_tiles(n, p.group);
        const PkRange keys(p, min(max(s - 1, 0), p.sequences - 1));
        return s >= 1 && s <= p.sequences ? PkParts(p.splits, p.part, p.causal != 0, p.group, n, keys.count).before(tiles) : tiles;
      });
    }
    rows = w.own * p.group;
    k_first = 0;
    m = 0;
    if (w.seq >= 0 && w.own > 0) {
      const PkRange keys(p, w.seq);
      k_first = keys.first;
      m = keys.count;
      if (shared) {
        const PkParts all(p.splits, p.part, p.causal != 0, p.group, w.own, m);
        if (counted) {  // the tile of the sequence's part w.tile: the last one before which no more parts lie
          int lo = 0, hi = pk_tiles(w.own, p.group);
          while (hi - lo > 1) {
            const int step = (hi - lo + 63) / 64, x = lo + lane * step;
            const int n = static_cast<int>(__popcll(__ballot(x < hi && all.before(x) <= w.tile)));
            lo += (n - 1) * step;
            hi = min(hi, lo + step);
          }
          split = w.tile - all.before(lo);
          w.tile = lo;
        }
        parts = all.of(w.tile);
      }
    }
    if (split >= parts) rows = 0;
    r0 = w.tile * kPkTile;
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
// reference score m and sum l. m starts at the first chunk's maximum (whose weight, the largest of a short
// row, is then 1 and rounds to itself) and moves when a chunk's exceeds it by 2^8.
template <typename T, int DT>
__global__ void __launch_bounds__(64 * kPkWaves, sizeof(T) == 2 ? (DT <= 32 ? 4 : DT <= 64 ? 3 : 2) : 1) pk_fwd_kernel(const PackParams p) {
  using Tile = PkTile<T, DT>;
  using Stream = PkStream<T, DT>;
  // arrays of their own, so that the compiler knows that the transfers under way do not write what it reads
  __shared__ __align__(16) unsigned char X0[Tile::BYTES], Y0[Tile::BYTES], X1[Tile::BYTES], Y1[Tile::BYTES];
  __shared__ uint32_t bad[2][2];  // pk_settle's rows of a chunk, by turns
  if (threadIdx.x < 4) bad[threadIdx.x >> 1][threadIdx.x & 1] = 0;
  constexpr int PF = sizeof(T) == 2 ? 3 : 2;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x >> 6)), grp = lane >> 5, col = lane & 31;
  const PkLane<T, DT> at(lane);
  const PkQueries w(p, lane, std::true_type());
  if (w.r0 >= w.rows) return;
  const int r1 = min(w.r0 + kPkTile, w.rows);
  T* out = static_cast<T*>(p.out);
  const int end = w.w.seq < 0 ? 0 : w.seen(p, r1 - 1), chunks = (end + kPkChunk - 1) / kPkChunk;  // that the workgroup sees
  const int parts = w.parts;
  if (p.splits > 1 && w.split == 0)  // one part writes its rows itself
    for (int r = w.r0 + static_cast<int>(threadIdx.x); r < r1; r += 64 * kPkWaves) p.part_n[w.stat(p, r)] = parts;
  if (w.w.seq < 0) {
    pk_zero_rows<T>(w.r0, r1, p.dim, [&](int r) { return w.row(p, out, kPkO, r); });
    return;
  }
  const int wr0 = w.r0 + 32 * wave, ri = wr0 + col;
  const bool valid = ri < w.rows;
  const int lim = valid ? w.seen(p, ri) : 0;
  const int wend = wr0 < w.rows ? w.seen(p, min(wr0 + 31, w.rows - 1)) : 0;  // keys that the wave sees
  const int wfull = wr0 + 31 < w.rows ? w.seen(p, wr0) : 0;                  // that every row of it sees
  const int all = w.seen(p, w.r0);                                           // that every row of the workgroup sees
  const bool few = wr0 < w.rows && w.seen(p, wr0) < kPkChunk, narrow = w.rows <= 32;
  const int per = (chunks + parts - 1) / parts, c0 = w.split * per, c1 = min(chunks, c0 + per);
  PkRow<T, DT> q;
  q.load(w.row(p, static_cast<const T*>(p.q), kPkQ, min(ri, w.rows - 1)), valid, p.dim, grp);
  const T* kp = static_cast<const T*>(p.k) + w.k_first * p.st[kPkK][0] + w.kv_head * p.st[kPkK][1];
  const T* vp = static_cast<const T*>(p.v) + w.k_first * p.st[kPkV][0] + w.kv_head * p.st[kPkV][1];
  float m = 0.0f, l = 0.0f;  // l: of the lane's half of the keys
  bool fresh = true;         // no key seen yet
  at_f16 o[DT / 32];
#pragma unroll
  for (int nd = 0; nd < DT / 32; ++nd) o[nd] = at_zero16();

  using Pair = typename Stream::Pair;
  auto tile = [&](unsigned char* K, unsigned char* V, int c) {  // behind the last: zeros, which nothing reads
    return Pair(K, kp, p.st[kPkK][0], V, vp, p.st[kPkV][0], c * kPkChunk, c < c1 ? w.m : 0, p.dim);
  };
  bool sick = false;  // pk_settle found some
  auto chunk = [&](unsigned char* Kb, unsigned char* Vb, int turn, int c, const Pair& next) {
    PkLds K = (PkLds)(Kb), V = (PkLds)(Vb);
    const int k0 = c * kPkChunk;
    if (min(k0 + kPkChunk, w.m) > all) {
      if (threadIdx.x < 2) bad[turn ^ 1][threadIdx.x] = 0;
      pk_settle<T, DT>(Vb, bad[turn]);
      sick = sick || pk_settled(bad[turn]) != 0;
    }
    if (k0 >= wend) {
      next.all();
      return;
    }
    at_f16 s0 = at_zero16(), s1 = at_zero16();
    if constexpr (sizeof(T) == 2) {
      // Phases of KS products: scores of keys 0 .. 31, of 32 .. 63 beside the softmax of the first, sums of
      // the first beside the softmax of the second, sums of the second. The vector work fits beside the
      // products of one wave; a CU's other workgroup fills the rest.
      using P = PkProducts<T, DT>;
      constexpr int KS = P::kScores, HA = KS >= 4 ? KS / 2 - 1 : 1, HB = KS - 1 - HA;  // steps up to the maximum, behind it
      float bm, alpha = 1.0f, late = 1.0f;  // late: what scales the first half's weights after their rounding
      // step t of the softmax of block x, whose keys start at k: x = scale2 s - m and its maximum, m moved if it
      // has to, weights and their sum (a lane sums its half of the keys until the end)
      auto soft = [&](at_f16& x, int k, auto step) {
        constexpr int t = decltype(step)::value, first = HB > 0 ? HA + 1 : HA, parts = HB > 0 ? HB : 1;
        if constexpr (t == 1) {
          if (k + 32 > wfull) pk_mask(x, k, lim, grp);
          bm = -INFINITY;
        }
        if constexpr (t >= 1 && t <= HA) {
          constexpr int lo = 16 * (t - 1) / HA, hi = 16 * t / HA;
          pk_for<hi - lo>([&](auto i) {
            x[lo + i] = fmaf(x[lo + i], p.scale2, -m);
            bm = fmaxf(bm, x[lo + i]);
          });
        }
        if constexpr (t == HA) {
          bm = at_max_halves(bm);
          const bool move = bm > kAtLazy || (fresh && bm != -INFINITY);
          if (__any(move)) {
            const float d = move ? bm : 0.0f, a = fresh ? 0.0f : at_exp2(-d);
            alpha *= a;
            m += d;
            l *= a;
            x -= d;
            fresh = fresh && !move;
          }
        }
        if constexpr (t >= first) {
          constexpr int lo = 16 * (t - first) / parts, hi = 16 * (t - first + 1) / parts;
          pk_for<hi - lo>([&](auto i) {
            x[lo + i] = at_exp2(x[lo + i]);
            l += x[lo + i];
          });
        }
      };
      auto rescale = [&](auto phase) {  // between phases: the sums of a phase belong to one m
        if (__any(alpha != 1.0f)) {
#pragma unroll
          for (int nd = 0; nd < DT / 32; ++nd) o[nd] *= alpha;
          if constexpr (phase == 2) late = alpha;
          alpha = 1.0f;
        }
      };
      typename P::Weights w0, w1;
      pk_pipe<4 * KS, PF>(
          [&](auto i) {
            constexpr int b = i / KS, t = i % KS;
            if constexpr (b < 2) return P::row_operand(K + b * 32 * Tile::ROW, at, t);
            else return P::sum_operand(V + (b - 2) * 32 * Tile::ROW, at, t);
          },
          [&](auto i, const auto& a) {
            constexpr int b = i / KS, t = i % KS;
            if constexpr (b == 0) P::score(s0, a, q, t);
            if constexpr (b == 1) P::score(s1, a, q, t);
            if constexpr (b == 2) P::sum(o, a, w0, t);
            if constexpr (b == 3) P::sum(o, a, w1, t);
          },
          [&](auto i) {
            constexpr int b = i / KS, t = i % KS;
            if constexpr (i < 2 * Stream::NV) next.template piece<i>();
            if constexpr (b == 1) soft(s0, k0, PkInt<t>{});
            if constexpr (b == 2) soft(s1, k0 + 32, PkInt<t>{});
            if constexpr ((b == 1 || b == 2) && t == KS - 1) {
              rescale(PkInt<b>{});
              if constexpr (b == 1) w0.set(s0);
              else w1.set(s1);
            }
          });
      // Rows of fewer than 64 keys, and sequences whose rows one wave holds: what the rounding of the weights left, too.
      // The rounding's errors do not average out over few keys, and delta, from the output, carries them into every ds
      // of the row, where they are as large as those of ds's own rounding. (60 calls of 1 to 8 sequences of 1 to 600
      // rows: 7 of 240 results were more than 1.5 times as far off as the exact ones rounded, with this and the same
      // for dq 1.) New tokens over caches are bound by the loads: 64 of them, 128 channels, are 1.00 times as far off as
      // the exact results rounded where it was 1.38, in 121 us for 116. For rows of every kind the products are half as
      // many again: 16,000 tokens of prompts 897 us for 631, to 1.00 from 1.2 to 1.4.
      if ((k0 == 0 && few) || narrow) pk_accumulate2<T, DT, 2>(o, V, pk_rest(s0) * late, o, V + 32 * Tile::ROW, pk_rest(s1), at);
    } else {
      next.all();
      pk_scores2<T, DT, PF>(s0, K, q, s1, K + 32 * Tile::ROW, q, at);
      if (k0 + kPkChunk > wfull) {
        pk_mask(s0, k0, lim, grp);
        pk_mask(s1, k0 + 32, lim, grp);
      }
      float bm = -INFINITY;
#pragma unroll
      for (int i = 0; i < 16; ++i) bm = fmaxf(bm, fmaxf(s0[i], s1[i]));
      bm = at_max_halves(bm) * p.scale2;
      if (bm != -INFINITY && (bm > m + kAtLazy || fresh)) {
        const float alpha = fresh ? 0.0f : at_exp2(m - bm);
        m = bm;
        l *= alpha;
        fresh = false;
#pragma unroll
        for (int nd = 0; nd < DT / 32; ++nd) o[nd] *= alpha;
      }
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        s0[i] = at_exp2(fmaf(s0[i], p.scale2, -m));
        s1[i] = at_exp2(fmaf(s1[i], p.scale2, -m));
        l += s0[i] + s1[i];
      }
      pk_accumulate2<T, DT, PF>(o, V, s0, o, V + 32 * Tile::ROW, s1, at);
    }
  };
  if (c0 < c1) tile(X0, Y0, c0).all();
  for (int c = c0; c < c1; c += 2) {
    pk_barrier();  // tile c is there, and every wave is done with tile c - 1
    chunk(X0, Y0, 0, c, tile(X1, Y1, c + 1));
    if (c + 1 >= c1) break;
    pk_barrier();
    chunk(X1, Y1, 1, c + 1, tile(X0, Y0, c + 2));
  }
  // Infinities and NaN of values: those that pk_settle took out, for the rows that see them, and those that the rest of a
  // weight, 0 or of either sign, made NaN. Where a row sees some in a channel, their sum is the result.
  bool odd = false;
  if constexpr (sizeof(T) == 2)
    if (few || narrow) {
#pragma unroll
      for (int nd = 0; nd < DT / 32; ++nd)
#pragma unroll
        for (int i = 0; i < 16; ++i) odd = odd || o[nd][i] != o[nd][i];
      odd = __any(odd);
    }
  if (sick || odd) {
    at_f16 y[DT / 32];
#pragma unroll
    for (int nd = 0; nd < DT / 32; ++nd) y[nd] = at_zero16();
#pragma unroll 1
    for (int j = (odd ? c0 : max(all / kPkChunk, c0)) * kPkChunk; j < min(c1 * kPkChunk, lim); ++j)
#pragma unroll
      for (int nd = 0; nd < DT / 32; ++nd)
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const int ch = 32 * nd + 8 * (i >> 2) + 4 * grp + (i & 3);
          float x = 0.0f;
          if (ch < p.dim) {
            if constexpr (sizeof(T) == 2) x = bf16_to_f32(vp[j * p.st[kPkV][0] + ch]);
            else x = vp[j * p.st[kPkV][0] + ch];
          }
          if (x - x != 0.0f) y[nd][i] += x;
        }
#pragma unroll
    for (int nd = 0; nd < DT / 32; ++nd)
#pragma unroll
      for (int i = 0; i < 16; ++i) o[nd][i] = y[nd][i] != 0.0f ? y[nd][i] : o[nd][i];
  }
  l = at_sum_halves(l);
  pk_barrier();  // the tiles hold the waves' scratch from here
  unsigned char* const scratch = (wave / 2 % 4 == 0 ? X0 : wave / 2 % 4 == 1 ? Y0 : wave / 2 % 4 == 2 ? X1 : Y1) + wave % 2 * (Tile::BYTES / 2);
  if (parts > 1) {  // sums as they are: registers hold 4 consecutive channels of the lane's row
    if (!valid) return;
    const int64_t part = static_cast<int64_t>(w.split) * p.q_rows * p.heads + w.stat(p, ri);
    float* po = p.part_o + part * p.dim;
#pragma unroll
    for (int nd = 0; nd < DT / 32; ++nd)
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const int ch = 32 * nd + 8 * c + 4 * grp;
        if (ch < p.dim) *reinterpret_cast<at_f4*>(po + ch) = at_f4{o[nd][4 * c], o[nd][4 * c + 1], o[nd][4 * c + 2], o[nd][4 * c + 3]};
      }
    if (grp == 0) *reinterpret_cast<float2*>(p.part_ml + part * 2) = float2{m, l};
    return;
  }
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;
  pk_store<T, DT>(o, inv, scratch, p.dim, lane, [&](int r) { return wr0 + r < w.rows ? w.row(p, out, kPkO, wr0 + r) : static_cast<T*>(nullptr); });
  if constexpr (sizeof(T) == 2) {
    T* rest = static_cast<T*>(p.rest);
    if (rest != nullptr)
      pk_store<T, DT, true>(o, inv, scratch, p.dim, lane,
                            [&](int r) { return wr0 + r < w.rows ? w.row(p, rest, kPkO, wr0 + r) : static_cast<T*>(nullptr); });
  }
  if (p.stats != nullptr && valid && grp == 0)
    *reinterpret_cast<float2*>(p.stats + 4 * w.stat(p, ri)) = pk_stats(m, l);
}

template <typename T>
__device__ __forceinline__ void pk_put4(T* to, at_f4 v) {
  if constexpr (sizeof(T) == 2) {
    *reinterpret_cast<uint2*>(to) = __builtin_bit_cast(uint2, __builtin_convertvector(v, pk_bf4));
  } else {
    *reinterpret_cast<at_f4*>(to) = v;
  }
}

// The split forward's parts joined, LPR lanes a row (token, head): each lane weighs some parts, then sums four
// channels at a time over all of them.
template <typename T, int LPR>
__global__ void __launch_bounds__(256) pk_join_kernel(const PackParams p) {
  const int64_t rows = static_cast<int64_t>(p.q_rows) * p.heads, row = static_cast<int64_t>(blockIdx.x) * (256 / LPR) + threadIdx.x / LPR;
  const int lane = threadIdx.x % LPR;
  const int parts = row < rows ? min(p.part_n[row], p.splits) : 0;
  float2 ml[kPkMostParts / LPR];  // of parts lane, lane + LPR, ..
  float m = -INFINITY, l = 0.0f;
#pragma unroll
  for (int i = 0; i < kPkMostParts / LPR; ++i) {
    const int s = lane + LPR * i;
    ml[i] = s < parts ? *reinterpret_cast<const float2*>(p.part_ml + (s * rows + row) * 2) : float2{0.0f, 0.0f};
    if (ml[i].y != 0.0f) m = fmaxf(m, ml[i].x);
  }
#pragma unroll
  for (int x = LPR / 2; x > 0; x /= 2) m = fmaxf(m, __shfl_xor(m, x, LPR));
#pragma unroll
  for (int i = 0; i < kPkMostParts / LPR; ++i) {
    ml[i].x = ml[i].y != 0.0f ? at_exp2(ml[i].x - m) : 0.0f;  // the part's weight
    l += ml[i].y * ml[i].x;
  }
#pragma unroll
  for (int x = LPR / 2; x > 0; x /= 2) l += __shfl_xor(l, x, LPR);
  if (parts <= 1) return;  // written already
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;
  const int64_t tok = row / p.heads, h = row - tok * p.heads;
  T* out = static_cast<T*>(p.out) + tok * p.st[kPkO][0] + h * p.st[kPkO][1];
  for (int ch = 4 * lane; ch < p.dim + 4 * (LPR - 1); ch += 4 * LPR) {  // every lane takes part in the shuffles
    const bool mine = ch < p.dim;
    at_f4 a = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int i = 0; i < kPkMostParts / LPR; ++i)
#pragma unroll 4
      for (int s = LPR * i; s < min(parts, LPR * (i + 1)); ++s) {
        const float w = __shfl(ml[i].x, s - LPR * i, LPR);
        if (mine && w != 0.0f) a += *reinterpret_cast<const at_f4*>(p.part_o + (s * rows + row) * p.dim + ch) * w;
      }
    if (!mine) continue;
    a *= inv;
    pk_put4(out + ch, a);
    if constexpr (sizeof(T) == 2)
      if (p.rest != nullptr)
        pk_put4(static_cast<T*>(p.rest) + (out - static_cast<T*>(p.out)) + ch, a - __builtin_convertvector(__builtin_convertvector(a, pk_bf4), at_f4));
  }
  if (p.stats != nullptr && lane == 0)
    *reinterpret_cast<float2*>(p.stats + 4 * row) = pk_stats(m, l);
}

// dq, and the rows' numbers for the key side (alone when gq is null).
template <typename T, int DT>
__global__ void __launch_bounds__(64 * kPkWaves, sizeof(T) == 2 ? (DT <= 64 ? 3 : 2) : 1) pk_bwd_q_kernel(const PackParams p) {
  using Tile = PkTile<T, DT>;
  using Stream = PkStream<T, DT>;
  // arrays of their own, so that the compiler knows that the transfers under way do not write what it reads
  __shared__ __align__(16) unsigned char X0[Tile::BYTES], Y0[Tile::BYTES], X1[Tile::BYTES], Y1[Tile::BYTES];
  __shared__ uint32_t bad[2][2];  // pk_settle's rows of a chunk, by turns
  if (threadIdx.x < 4) bad[threadIdx.x >> 1][threadIdx.x & 1] = 0;
  constexpr int PF = sizeof(T) == 2 ? 3 : 2;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x >> 6)), grp = lane >> 5, col = lane & 31;
  const PkLane<T, DT> at(lane);
  const PkQueries w(p, lane, std::false_type());
  if (w.r0 >= w.rows) return;
  const int r1 = min(w.r0 + kPkTile, w.rows);
  T* gq = static_cast<T*>(p.gq);
  if (w.w.seq < 0) {
    if (gq != nullptr) pk_zero_rows<T>(w.r0, r1, p.dim, [&](int r) { return w.row(p, gq, kPkGQ, r); });
    return;
  }
  const int wr0 = w.r0 + 32 * wave, ri = wr0 + col, rc = min(ri, w.rows - 1);
  const bool valid = ri < w.rows;
  const int lim = valid ? w.seen(p, ri) : 0;
  const int end = w.seen(p, r1 - 1);
  const int wend = wr0 < w.rows ? w.seen(p, min(wr0 + 31, w.rows - 1)) : 0;
  const int wfull = wr0 + 31 < w.rows ? w.seen(p, wr0) : 0;
  const int all = w.seen(p, w.r0);  // keys that every row of the workgroup sees
  const bool few = wr0 < w.rows && w.seen(p, wr0) < kPkChunk;
  const int chunks = (end + kPkChunk - 1) / kPkChunk;
  PkRow<T, DT> q, go;
  q.load(w.row(p, static_cast<const T*>(p.q), kPkQ, rc), valid, p.dim, grp);
  go.load(w.row(p, static_cast<const T*>(p.go), kPkGO, rc), valid, p.dim, grp);
  float m, ll, delta;
  {
    PkRow<T, DT> o;
    o.load(w.row(p, static_cast<const T*>(p.o), kPkO, rc), valid, p.dim, grp);
    delta = go.dot(o);
    if constexpr (sizeof(T) == 2) {
      // with what out's rounding left: delta's error from the rounding would be as large as that of ds's own
      // (packed training, error of grad_q and grad_k against f64: 2.6e-3 without, 2.4e-3 with it)
      if (p.rest != nullptr) {
        o.load(w.row(p, static_cast<const T*>(p.rest), kPkO, rc), valid, p.dim, grp);
        delta += go.dot(o);
      }
    }
    delta = at_sum_halves(delta);
    const int64_t row = 4 * w.stat(p, rc);
    m = p.stats[row];
    ll = p.stats[row + 1];
    // for the key side: delta; bf16: -delta and -(m + log2 l) / scale2, which its sums start from (the weight is
    // 2^(scale2 s) then; the number is rounded at its own size, 2^-24 of it)
    if (p.numbers != nullptr && valid && grp == 0)
      *reinterpret_cast<at_f4*>(p.numbers + row) = sizeof(T) == 2 ? at_f4{m, ll, -delta, -(m + ll) / p.scale2} : at_f4{m, ll, delta, 0.0f};
  }
  if (gq == nullptr) return;
  constexpr bool bf = sizeof(T) == 2;
  if (bf) m += ll;  // rounded at its own size, 2^-24 of it
  const T* kp = static_cast<const T*>(p.k) + w.k_first * p.st[kPkK][0] + w.kv_head * p.st[kPkK][1];
  const T* vp = static_cast<const T*>(p.v) + w.k_first * p.st[kPkV][0] + w.kv_head * p.st[kPkV][1];
  at_f16 dq[DT / 32];
#pragma unroll
  for (int nd = 0; nd < DT / 32; ++nd) dq[nd] = at_zero16();

  using Pair = typename Stream::Pair;
  auto tile = [&](unsigned char* K, unsigned char* V, int c) {  // behind the last: zeros, which nothing reads
    return Pair(K, kp, p.st[kPkK][0], V, vp, p.st[kPkV][0], c * kPkChunk, c < chunks ? w.m : 0, p.dim);
  };
  float factor = p.scale;  // NaN: the row sees a key that is not finite
  auto chunk = [&](unsigned char* Kb, unsigned char* Vb, int turn, int c, const Pair& next) {
    PkLds K = (PkLds)(Kb), V = (PkLds)(Vb);
    const int k0 = c * kPkChunk;
    if (min(k0 + kPkChunk, w.m) > all) {
      if (threadIdx.x < 2) bad[turn ^ 1][threadIdx.x] = 0;
      pk_settle<T, DT>(Kb, bad[turn]);
      const uint64_t sick = pk_settled(bad[turn]);
      if (sick != 0 && k0 + static_cast<int>(__builtin_ctzll(sick)) < lim) factor = NAN;
    }
    if (k0 >= wend) {
      next.all();
      return;
    }
    if constexpr (bf) {
      // Phases of KS products: S, dP beside the weights, of the first 32 keys and of the second (beside ds of the
      // first), then their sums (beside ds of the second).
      using P = PkProducts<T, DT>;
      constexpr int KS = P::kScores;
      at_f16 sa = at_zero16(), sb = at_zero16(), da = at_zero16(), db = at_zero16();
      typename P::Weights wa, wb;
      PkLane<T, DT> now = at;  // as in pk_bwd_kv_kernel
      asm volatile("" : "+v"(now.row), "+v"(now.tr));
      auto weigh = [&](at_f16& s, auto t) { pk_beside<KS, t>([&](int i) { s[i] = at_exp2(fmaf(s[i], p.scale2, -m)); }); };
      auto slope = [&](at_f16& s, const at_f16& d, typename P::Weights& w, int k, auto t) {
        pk_beside<KS, t>([&](int i) { s[i] *= d[i] - delta; });
        if constexpr (t == KS - 1) {
          if (k + 32 > wfull) {
#pragma unroll
            for (int i = 0; i < 16; ++i) s[i] = k + 8 * (i >> 2) + 4 * grp + (i & 3) < lim ? s[i] : 0.0f;
          }
          w.set(s);
        }
      };
      pk_pipe<6 * KS, PF>(
          [&](auto i) {
            constexpr int b = i / KS, t = i % KS;
            const PkLds X = (b == 1 || b == 3 ? V : K) + (b == 2 || b == 3 || b == 5 ? 32 * Tile::ROW : 0);
            if constexpr (b < 4) return P::row_operand(X, now, t);
            else return P::sum_operand(X, now, t);
          },
          [&](auto i, const auto& a) {
            constexpr int b = i / KS, t = i % KS;
            if constexpr (b == 0) P::score(sa, a, q, t);
            if constexpr (b == 1) P::score(da, a, go, t);
            if constexpr (b == 2) P::score(sb, a, q, t);
            if constexpr (b == 3) P::score(db, a, go, t);
            if constexpr (b == 4) P::sum(dq, a, wa, t);
            if constexpr (b == 5) P::sum(dq, a, wb, t);
          },
          [&](auto i) {
            constexpr int b = i / KS;
            constexpr PkInt<i % KS> t{};
            if constexpr (i < 2 * Stream::NV) next.template piece<i>();
            if constexpr (b == 1) weigh(sa, t);
            if constexpr (b == 2) slope(sa, da, wa, k0, t);
            if constexpr (b == 3) weigh(sb, t);
            if constexpr (b == 4) slope(sb, db, wb, k0 + 32, t);
          });
      if (k0 == 0 && few)  // as in the forward: of ds
        pk_accumulate2<T, DT, 2>(dq, K, pk_rest(sa), dq, K + 32 * Tile::ROW, pk_rest(sb), now);
    } else {
      next.all();
#pragma unroll 1
      for (int h = 0; h < kPkChunk; h += 32) {
        at_f16 s = at_zero16(), dp = at_zero16();
        pk_scores2<T, DT, PF>(s, K + h * Tile::ROW, q, dp, V + h * Tile::ROW, go, at);
#pragma unroll
        for (int i = 0; i < 16; ++i) s[i] = at_exp2(fmaf(s[i], p.scale2, -m) - ll) * (dp[i] - delta);
        if (k0 + h + 32 > wfull) {
#pragma unroll
          for (int i = 0; i < 16; ++i) s[i] = k0 + h + 8 * (i >> 2) + 4 * grp + (i & 3) < lim ? s[i] : 0.0f;
        }
        pk_accumulate<T, DT, PF>(dq, K + h * Tile::ROW, s, at);
      }
    }
  };
  if (chunks > 0) tile(X0, Y0, 0).all();
  for (int c = 0; c < chunks; c += 2) {
    pk_barrier();
    chunk(X0, Y0, 0, c, tile(X1, Y1, c + 1));
    if (c + 1 >= chunks) break;
    pk_barrier();
    chunk(X1, Y1, 1, c + 1, tile(X0, Y0, c + 2));
  }
  pk_barrier();
  unsigned char* const scratch = (wave / 2 % 4 == 0 ? X0 : wave / 2 % 4 == 1 ? Y0 : wave / 2 % 4 == 2 ? X1 : Y1) + wave % 2 * (Tile::BYTES / 2);
  pk_store<T, DT>(dq, factor, scratch, p.dim, lane,
                  [&](int r) { return wr0 + r < w.rows ? w.row(p, gq, kPkGQ, wr0 + r) : static_cast<T*>(nullptr); });
}

// ---- keys on their own side: dk and dv ---------------------------------------------------------

struct PkKeys {
  PkPlace w;
  int kv_head, part;
  int b0, b1;            // keys of the tile, in the sequence's range
  int m, n, q_first;     // keys and queries of the sequence, its first query row
  int shift;
  int first, chunks;     // the first token that sees a key of the tile; chunks of tokens from there
  int parts;             // workgroups that share them
  // b: tile and key head (fastest, as in PkQueries; the first tiles, which the most queries of a causal sequence
  // see, first)
  __device__ PkKeys(const PackParams& p, const PkRows& walk, int lane, int b, int part_) : part(part_) {
    const int slot = b / p.kv_heads;
    kv_head = b - slot * p.kv_heads;
    w = pk_place<false>(p.k_offsets, p.sequences, p.k_rows, 1, pk_line(slot, p.slots, p.kv_heads), p.slots, lane, false, [](int, int n) { return pk_tiles(n, 1); });
    b0 = w.tile * kPkTile;
    b1 = min(b0 + kPkTile, w.own);
    m = n = q_first = 0;
    if (w.seq >= 0) {
      m = p.k_lengths != nullptr ? min(max(p.k_lengths[w.seq], 0), w.own) : w.own;
      q_first = min(max(p.q_offsets[w.seq], 0), p.q_rows);
      n = min(max(p.q_offsets[w.seq + 1], q_first), p.q_rows) - q_first;
    }
    shift = m - n;
    first = p.causal ? min(max(b0 - shift, 0), n) : 0;
    chunks = b0 < m ? (n - first + walk.tokens - 1) / walk.tokens : 0;
    parts = min(max((chunks + kPkPart - 1) / kPkPart, 1), p.splits);
  }
  template <typename T>
  __device__ T* row(const PackParams& p, T* base, int t, int j) const {
    return base + (static_cast<int64_t>(w.first) + j) * p.st[t][0] + kv_head * p.st[t][1];
  }
  // row of the parts' sums of key j
  __device__ int64_t part_row(const PackParams& p, int which, int j) const {
    return (static_cast<int64_t>(which) * p.k_rows + w.first + j) * p.kv_heads + kv_head;
  }
};

// A workgroup takes 128 keys, 32 a wave in registers, and walks over the rows (tokens and heads of the key
// head's group) that see them, 64 at a time. A tile that many rows see is shared by several workgroups,
// whose sums pk_join_kv_kernel adds in their order.
template <typename T, int DT>
__global__ void __launch_bounds__(64 * kPkWaves, sizeof(T) == 2 ? (DT <= 64 ? 3 : 2) : 1) pk_bwd_kv_kernel(const PackParams p) {
  using Tile = PkTile<T, DT>;
  using Stream = PkStream<T, DT>;
  // arrays of their own, so that the compiler knows that the transfers under way do not write what it reads
  __shared__ __align__(16) unsigned char X0[Tile::BYTES], Y0[Tile::BYTES], X1[Tile::BYTES], Y1[Tile::BYTES];
  __shared__ uint32_t bad[2][2];  // pk_settle's rows of a chunk, by turns
  if (threadIdx.x < 4) bad[threadIdx.x >> 1][threadIdx.x & 1] = 0;
  // of the tile's rows: the numbers that its scores and dP start from (bf16), or m, log2 l and delta (f32);
  // the keys that the row sees
  __shared__ __align__(16) float row_s[2][kPkChunk], row_d[2][kPkChunk], row_l[2][sizeof(T) == 2 ? 4 : kPkChunk];
  __shared__ __align__(16) int row_lim[2][kPkChunk];
  constexpr bool bf = sizeof(T) == 2;
  constexpr int PF = bf && DT != 64 && DT != 128 ? 3 : 2;
  // At 128 channels k, v, dk and dv take 192 of a wave's 256 registers. The last KEEP pieces of v wait in LDS: in
  // registers the compiler spilled them, and each reload from scratch memory waited for the tile in flight. Three
  // registers of other values are spilled still, two of them read back in the loop, behind a chunk's products.
  constexpr int KEEP = bf && DT == 128 ? 3 : 0;
  __shared__ __align__(16) unsigned char kept_rows[KEEP > 0 ? KEEP * kPkWaves * 1024 : 16];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x >> 6)), grp = lane >> 5, col = lane & 31;
  const PkRows walk(p.group);
  // the parts of a tile are a grid of tiles apart, the last of all tiles first: of shared tiles all parts are full,
  // those of one part, down to a few rows, come last and even out
  const int tiles = static_cast<int>(gridDim.x) / p.splits, turn = static_cast<int>(blockIdx.x) / tiles;
  const PkKeys w(p, walk, lane, static_cast<int>(blockIdx.x) - turn * tiles, p.splits - 1 - turn);
  if (w.b0 >= w.w.own || w.part >= w.parts) return;
  T* gk = static_cast<T*>(p.gk);
  T* gv = static_cast<T*>(p.gv);
  if (w.chunks <= 0) {
    if (gk != nullptr) pk_zero_rows<T>(w.b0, w.b1, p.dim, [&](int j) { return w.row(p, gk, kPkGK, j); });
    if (gv != nullptr) pk_zero_rows<T>(w.b0, w.b1, p.dim, [&](int j) { return w.row(p, gv, kPkGV, j); });
    return;
  }
  const int m = w.m, shift = w.shift;
  const int wb0 = w.b0 + 32 * wave;
  PkRow<T, DT> k, v;
  {
    const int kj = wb0 + col;
    k.load(w.row(p, static_cast<const T*>(p.k), kPkK, min(kj, m - 1)), kj < m, p.dim, grp);
    v.load(w.row(p, static_cast<const T*>(p.v), kPkV, min(kj, m - 1)), kj < m, p.dim, grp);
  }
  if constexpr (KEEP > 0)  // of this lane, so no barrier
    for (int j = 0; j < KEEP; ++j) *reinterpret_cast<at_bf8*>(kept_rows + threadIdx.x * 16 + j * kPkWaves * 1024) = v.x[DT / 16 - KEEP + j];
  const T* qp = static_cast<const T*>(p.q) + w.q_first * p.st[kPkQ][0] + static_cast<int64_t>(w.kv_head) * p.group * p.st[kPkQ][1];
  const T* gp = static_cast<const T*>(p.go) + w.q_first * p.st[kPkGO][0] + static_cast<int64_t>(w.kv_head) * p.group * p.st[kPkGO][1];
  const float* sp = p.numbers + 4 * (static_cast<int64_t>(w.q_first) * p.heads + w.kv_head * p.group);
  const int per = (w.chunks + w.parts - 1) / w.parts, c0 = w.part * per, c1 = min(w.chunks, c0 + per);
  at_f16 dk[DT / 32], dv[DT / 32];
#pragma unroll
  for (int nd = 0; nd < DT / 32; ++nd) dk[nd] = dv[nd] = at_zero16();

  const int sq[2] = {static_cast<int>(p.st[kPkQ][0] * static_cast<int>(sizeof(T))), static_cast<int>(p.st[kPkQ][1] * static_cast<int>(sizeof(T)))};
  const int sg[2] = {static_cast<int>(p.st[kPkGO][0] * static_cast<int>(sizeof(T))), static_cast<int>(p.st[kPkGO][1] * static_cast<int>(sizeof(T)))};
  // Tile c into Q, G and the row arrays `buf`: the rows' numbers by one wave each, a row a lane.
  auto stage = [&](unsigned char* Q, unsigned char* G, int buf, int c) {
    const int t0 = w.first + c * walk.tokens, count = min(walk.tokens, w.n - t0) * p.group;
    int thread = threadIdx.x;
    asm volatile("" : "+v"(thread));  // the pieces' offsets are formed anew (as in block)
    const __amdgpu_buffer_rsrc_t qs = pk_buffer(qp + t0 * p.st[kPkQ][0], kPkFar), gs = pk_buffer(gp + t0 * p.st[kPkGO][0], kPkFar);
#pragma unroll
    for (int v = 0; v < Stream::NV; ++v) {
      const int x = Stream::row(thread, v), t = walk.token(x), g = x - t * p.group, ch = Stream::channel(thread, v);
      const bool ok = x < count && (p.dim == Tile::DP || ch < p.dim);
      Stream::transfer(qs, ok ? t * sq[0] + g * sq[1] + ch * static_cast<int>(sizeof(T)) : kPkFar, Q, v);
      Stream::transfer(gs, ok ? t * sg[0] + g * sg[1] + ch * static_cast<int>(sizeof(T)) : kPkFar, G, v);
    }
    const int x = thread & 63, t = walk.token(x), g = x - t * p.group, o = x < count ? (t * p.heads + g) * 16 : kPkFar;
    const __amdgpu_buffer_rsrc_t ss = pk_buffer(sp + 4 * static_cast<int64_t>(t0) * p.heads, kPkFar);
    if (wave == 0) __builtin_amdgcn_raw_ptr_buffer_load_lds(ss, (MSDA_LDS void*)(row_s[buf]), 4, o + (bf ? 12 : 0), 0, 0, 0);
    if (wave == 1) __builtin_amdgcn_raw_ptr_buffer_load_lds(ss, (MSDA_LDS void*)(row_d[buf]), 4, o + 8, 0, 0, 0);
    if (wave == 2 && !bf) __builtin_amdgcn_raw_ptr_buffer_load_lds(ss, (MSDA_LDS void*)(row_l[buf]), 4, o + 4, 0, 0, 0);
    if (wave == 3) row_lim[buf][x] = x >= count ? 0 : p.causal ? min(max(t0 + t + shift + 1, 0), m) : m;
  };
  // One 32-row block; `all`: every row sees every key of the wave.
  auto block = [&](bool all, PkLds Q, PkLds G, int h, const float* rs, const float* rd, const float* rl, const int* lims) {
    // All that a lane's place gives is formed anew in each block, the operands' offsets in each phase: kept, they spill
    // at 128 channels.
    int thread = threadIdx.x;
    asm volatile("" : "+v"(thread));
    const int lane = thread & 63, grp = lane >> 5, col = lane & 31;
    PkLane<T, DT> now(lane);
    now.row += h * Tile::ROW;
    now.tr += h * Tile::ROW;
    asm volatile("" : "+v"(now.row), "+v"(now.tr));
    // bf16: the matrix units start from the rows' numbers
    auto start = [&](at_f16& x, const float* numbers) {
#pragma unroll
      for (int c4 = 0; c4 < 4; ++c4) {
        const at_f4 a = bf ? *reinterpret_cast<const at_f4*>(numbers + 8 * c4 + 4 * grp) : at_f4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int j = 0; j < 4; ++j) x[4 * c4 + j] = a[j];
      }
    };
    uint32_t kept = static_cast<uint32_t>(reinterpret_cast<uintptr_t>((MSDA_LDS unsigned char*)(kept_rows))) + thread * 16;
    asm volatile("" : "+v"(kept));  // one register: the arrays' addresses do not fit an LDS instruction's offset
    at_f16 s, dp;
    start(s, rs);
    if (!bf) start(dp, rd);
    using P = PkProducts<T, DT>;
    const int kj = wb0 + col;
    auto unseen = [&](at_f16& x) {  // pairs that are not seen weigh nothing
      if (all) return;
#pragma unroll
      for (int c4 = 0; c4 < 4; ++c4) {
        const int4 lm = *reinterpret_cast<const int4*>(lims + 8 * c4 + 4 * grp);
        x[4 * c4] = kj < lm.x ? x[4 * c4] : 0.0f;
        x[4 * c4 + 1] = kj < lm.y ? x[4 * c4 + 1] : 0.0f;
        x[4 * c4 + 2] = kj < lm.z ? x[4 * c4 + 2] : 0.0f;
        x[4 * c4 + 3] = kj < lm.w ? x[4 * c4 + 3] : 0.0f;
      }
    };
    if constexpr (bf) {
      // Phases of KS products: S, dP beside the weights, dv beside ds, dk.
      constexpr int KS = P::kScores;
      typename P::Weights w, ds;
      at_bf8 last[KEEP > 0 ? KEEP : 1];
      pk_pipe<4 * KS, PF>(
          [&](auto i) {
            constexpr int b = i / KS, t = i % KS;
            const PkLds X = b == 0 || b == 3 ? Q : G;
            if constexpr (t == 0) asm volatile("" : "+v"(now.row), "+v"(now.tr));
            if constexpr (b < 2) return P::row_operand(X, now, t);
            else return P::sum_operand(X, now, t);
          },
          [&](auto i, const auto& a) {
            constexpr int b = i / KS, t = i % KS;
            if constexpr (b == 0) P::score(s, a, k, t);
            if constexpr (b == 1 && t < KS - KEEP) P::score(dp, a, v, t);
            if constexpr (b == 1 && t >= KS - KEEP) P::score(dp, a, last[t - (KS - KEEP)]);
            if constexpr (b == 2) P::sum(dv, a, w, t);
            if constexpr (b == 3) P::sum(dk, a, ds, t);
          },
          [&](auto i) {
            constexpr int b = i / KS, t = i % KS;
            if constexpr (i == KS - 1) start(dp, rd);
            if constexpr (KEEP > 0 && b == 1 && t + 2 >= KS - KEEP && t + 2 < KS)
              last[t + 2 - (KS - KEEP)] = *reinterpret_cast<const MSDA_LDS at_bf8*>(reinterpret_cast<PkLds>(static_cast<uintptr_t>(kept)) + (t + 2 - (KS - KEEP)) * kPkWaves * 1024);
            if constexpr (b == 1) pk_beside<KS, t>([&](int j) { s[j] = at_exp2(s[j] * p.scale2); });
            if constexpr (b == 1 && t == KS - 1) {
              unseen(s);
              w.set(s);
            }
            if constexpr (b == 2) pk_beside<KS, t>([&](int j) { dp[j] *= s[j]; });
            if constexpr (b == 2 && t == KS - 1) {
              unseen(dp);
              ds.set(dp);
            }
          });
    } else {
      pk_scores2<T, DT, PF>(s, Q, k, dp, G, v, now);
#pragma unroll
      for (int c4 = 0; c4 < 4; ++c4) {
        const int a = 8 * c4 + 4 * grp;
        const at_f4 mm = *reinterpret_cast<const at_f4*>(rs + a), ll = *reinterpret_cast<const at_f4*>(rl + a);
        const at_f4 dd = *reinterpret_cast<const at_f4*>(rd + a);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int i = 4 * c4 + j;
          s[i] = at_exp2(fmaf(s[i], p.scale2, -mm[j]) - ll[j]);
          dp[i] = s[i] * (dp[i] - dd[j]);
        }
      }
      unseen(s);
      unseen(dp);
      pk_accumulate2<T, DT, PF>(dv, G, s, dk, Q, dp, now);
    }
  };
  bool spoilt = false;  // the lane's key is seen by a row that is not finite
  auto settle = [&](unsigned char* Q, unsigned char* G, int buf, int c) {
    const int t0 = w.first + c * walk.tokens;
    if (!p.causal || t0 + shift >= min(w.b1, m) - 1) return;  // every row sees every key
    if (threadIdx.x < 2) bad[buf ^ 1][threadIdx.x] = 0;
    pk_settle<T, DT>(Q, bad[buf]);
    pk_settle<T, DT>(G, bad[buf]);
    const uint64_t sick = pk_settled(bad[buf]);
    // rows see more keys the later they come
    if (sick != 0) spoilt = spoilt || wb0 + col < row_lim[buf][63 - static_cast<int>(__builtin_clzll(sick))];
  };
  auto chunk = [&](const unsigned char* Qb, const unsigned char* Gb, int buf, int c) {
    PkLds Q = (PkLds)(Qb), G = (PkLds)(Gb);
    const int t0 = w.first + c * walk.tokens, t1 = min(t0 + walk.tokens, w.n), count = (t1 - t0) * p.group;
    if (wb0 >= m || (p.causal && t1 + shift <= wb0)) return;
    // every row sees every key of the wave
    const bool full = __builtin_amdgcn_readfirstlane(count == kPkChunk && wb0 + 32 <= m && (!p.causal || t0 + shift >= wb0 + 31)) != 0;
#pragma unroll 1
    for (int h = 0; h < count; h += 32)
      block(full, Q, G, h, row_s[buf] + h, row_d[buf] + h, row_l[buf] + (bf ? 0 : h), row_lim[buf] + h);
  };
  if (c0 < c1) stage(X0, Y0, 0, c0);
  for (int c = c0; c < c1; c += 2) {
    pk_barrier();
    settle(X0, Y0, 0, c);
    if (c + 1 < c1) stage(X1, Y1, 1, c + 1);
    chunk(X0, Y0, 0, c);
    if (c + 1 >= c1) break;
    pk_barrier();
    settle(X1, Y1, 1, c + 1);
    if (c + 2 < c1) stage(X0, Y0, 0, c + 2);
    chunk(X1, Y1, 1, c + 1);
  }
  pk_barrier();
  if (__any(spoilt || wb0 + col >= m)) {  // keys from m on (rows of the range behind the sequence's keys) get zeros
    const float none = spoilt ? NAN : 0.0f;
    const bool keep = !spoilt && wb0 + col < m;
#pragma unroll
    for (int nd = 0; nd < DT / 32; ++nd)
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        dk[nd][i] = keep ? dk[nd][i] : none;
        dv[nd][i] = keep ? dv[nd][i] : none;
      }
  }
  if (w.parts > 1) {
    const int kj = wb0 + col;
    if (kj >= w.b1) return;
    float* pk = p.part_kv + w.part_row(p, 2 * w.part, kj) * p.dim;
    float* pv = p.part_kv + w.part_row(p, 2 * w.part + 1, kj) * p.dim;
#pragma unroll
    for (int nd = 0; nd < DT / 32; ++nd)
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const int ch = 32 * nd + 8 * c + 4 * grp;
        if (ch >= p.dim) continue;
        *reinterpret_cast<at_f4*>(pk + ch) = at_f4{dk[nd][4 * c], dk[nd][4 * c + 1], dk[nd][4 * c + 2], dk[nd][4 * c + 3]};
        *reinterpret_cast<at_f4*>(pv + ch) = at_f4{dv[nd][4 * c], dv[nd][4 * c + 1], dv[nd][4 * c + 2], dv[nd][4 * c + 3]};
      }
    return;
  }
  unsigned char* const scratch = (wave / 2 % 4 == 0 ? X0 : wave / 2 % 4 == 1 ? Y0 : wave / 2 % 4 == 2 ? X1 : Y1) + wave % 2 * (Tile::BYTES / 2);
  if (gk != nullptr)
    pk_store<T, DT>(dk, p.scale, scratch, p.dim, lane, [&](int r) { return wb0 + r < w.b1 ? w.row(p, gk, kPkGK, wb0 + r) : static_cast<T*>(nullptr); });
  if (gv != nullptr)
    pk_store<T, DT>(dv, 1.0f, scratch, p.dim, lane, [&](int r) { return wb0 + r < w.b1 ? w.row(p, gv, kPkGV, wb0 + r) : static_cast<T*>(nullptr); });
}

// The sums of a tile's parts, in their order: kPkJoin workgroups a tile, of all key heads (which have as many parts).
template <typename T>
__global__ void __launch_bounds__(256) pk_join_kv_kernel(const PackParams p) {
  const int tile = static_cast<int>(blockIdx.x) / kPkJoin, share = kPkTile / kPkJoin;
  PkKeys w(p, PkRows(p.group), threadIdx.x & 63, tile * p.kv_heads, 0);
  if (w.parts == 1) return;
  const int first = w.b0 + share * (static_cast<int>(blockIdx.x) % kPkJoin), keys = min(share, w.b1 - first), pieces = p.dim / 4;
  for (int i = threadIdx.x; i < 2 * keys * p.kv_heads * pieces; i += 256) {
    const int r = i / pieces, ch = 4 * (i - r * pieces), row = r >> 1, which = r & 1, key = row / p.kv_heads;
    w.kv_head = row - key * p.kv_heads;
    T* base = static_cast<T*>(which == 0 ? p.gk : p.gv);
    if (base == nullptr) continue;
    at_f4 a = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 4
    for (int s = 0; s < w.parts; ++s) a += *reinterpret_cast<const at_f4*>(p.part_kv + w.part_row(p, 2 * s + which, first + key) * p.dim + ch);
    pk_put4(w.row(p, base, which == 0 ? kPkGK : kPkGV, first + key) + ch, which == 0 ? a * p.scale : a);
  }
}

}  // namespace msda
