// cache4_kernels.h — gfx950 device code for a cache of keys and values in 4 bits: writing new rows into it, reading
// rows back, and softmax attention of few query rows over it. (Many rows a sequence: packed_attention_kernels.h's
// forward, whose tiles are filled from the cache by PkCachePair.) The numbers: cache4_common.h.
//
// Layout. codes [kv_heads][rows][16 B], scales [kv_heads][rows][B] with B = ceil(head_dim / 32): head-major, so that the
// rows of one head are one stream of whole lines (row-major, 64 bytes of a row would be half of a 128-byte line).
#pragma once

#include "cache4_common.h"
#include "packed_attention_kernels.h"
#include "rotary_kernels.h"  // rot_load, rot_store

namespace msda {

// ---- writing and reading rows ------------------------------------------------------------------

struct Cache4Params {
  const void* x[2];   // new keys, values [tokens, kv_heads, dim] (write)
  void* y[2];         // the same (read)
  uint8_t* codes[2];  // of keys, values
  uint8_t* scales[2];
  int64_t st[2][2];   // element strides (token, head) of x or y
  const int32_t* q_offsets;
  const int32_t* k_offsets;
  const int32_t* k_lengths;  // or null
  int sequences, tokens, rows, kv_heads, dim, blocks;
};

// The cache row of token t, the newest of its sequence's keys being its last token's; -1: none. By the whole wave.
__device__ __forceinline__ int64_t c4_row(const Cache4Params& p, int t, int lane) {
  // the last sequence that starts at t or before, 64 offsets at a time
  int lo = 0, hi = p.sequences + 1;
  while (hi - lo > 1) {
    const int step = (hi - lo + 63) / 64, x = lo + lane * step;
    const int n = static_cast<int>(__popcll(__ballot(x < hi && p.q_offsets[min(x, p.sequences)] <= t)));
    if (n == 0) return -1;
    lo += (n - 1) * step;
    hi = min(hi, lo + step);
  }
  if (lo >= p.sequences) return -1;
  const int q0 = p.q_offsets[lo], q1 = p.q_offsets[lo + 1];
  if (t < q0 || t >= q1) return -1;
  const int first = min(max(p.k_offsets[lo], 0), p.rows), end = min(max(p.k_offsets[lo + 1], first), p.rows);
  const int m = p.k_lengths != nullptr ? min(max(p.k_lengths[lo], 0), end - first) : end - first;
  const int64_t place = static_cast<int64_t>(m) - (static_cast<int64_t>(q1) - t);
  return place >= 0 ? first + place : -1;
}

// A lane's 8 channels: tensor, head, block and quarter of it from its number among the token's.
struct C4Unit {
  int which, head, block, quarter;
  __device__ __forceinline__ C4Unit(const Cache4Params& p, int u) {
    quarter = u & 3;
    const int row = u >> 2, heads = row / p.blocks;
    block = row - heads * p.blocks;
    which = heads >= p.kv_heads ? 1 : 0;
    head = heads - which * p.kv_heads;
  }
  __device__ __forceinline__ int channel() const { return 32 * block + 8 * quarter; }
};

// A wave takes 64 units of one token; the four lanes of a block find its maximum together. Bound by the bytes of the new
// rows (11,931 tokens of 8 heads, 128 channels, f32: 111 MB in 22 us, 4.9 TB/s).
template <typename T>
__global__ void __launch_bounds__(256) cache4_write_kernel(const Cache4Params p) {
  const int lane = static_cast<int>(threadIdx.x) & 63, units = 2 * p.kv_heads * p.blocks * 4, waves = (units + 63) / 64;
  const int64_t index = static_cast<int64_t>(blockIdx.x) * 4 + __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x >> 6));
  const int t = static_cast<int>(index / waves);
  if (t >= p.tokens) return;
  const int u = static_cast<int>(index - static_cast<int64_t>(t) * waves) * 64 + lane;
  const C4Unit at(p, min(u, units - 1));
  const int ch = at.channel();
  float v[8] = {};
  if (ch < p.dim) {
    const T* x = static_cast<const T*>(p.x[at.which]) + static_cast<int64_t>(t) * p.st[at.which][0] + at.head * p.st[at.which][1] + ch;
    constexpr int E = 16 / static_cast<int>(sizeof(T));
#pragma unroll
    for (int j = 0; j < 8; j += E) rot_load<T>(v + j, x + j);
  }
  const int64_t row = c4_row(p, t, lane);
  uint32_t most = 0;  // as an integer: NaN above infinity above all numbers
#pragma unroll
  for (int j = 0; j < 8; ++j) most = max(most, __float_as_uint(v[j]) & 0x7fffffffu);
  most = max(most, static_cast<uint32_t>(__shfl_xor(static_cast<int>(most), 1)));
  most = max(most, static_cast<uint32_t>(__shfl_xor(static_cast<int>(most), 2)));
  if (row < 0 || u >= units) return;
  const bool bad = most >= 0x7f800000u;
  // 1.75 2^k and less is 7 2^(k - 2) at most: the exponent goes up one behind it
  const int e = min(max(static_cast<int>((most + 0x1fffffu) >> 23) - 129, -120), 125);
  const float inverse = __uint_as_float(static_cast<uint32_t>(127 - e) << 23);
  uint32_t codes = 0;
  codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, v[0] * inverse, v[1] * inverse, 1.0f, 0);
  codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, v[2] * inverse, v[3] * inverse, 1.0f, 1);
  codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, v[4] * inverse, v[5] * inverse, 1.0f, 2);
  codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, v[6] * inverse, v[7] * inverse, 1.0f, 3);
  const int64_t block = (at.head * static_cast<int64_t>(p.rows) + row) * p.blocks + at.block;
  *reinterpret_cast<uint32_t*>(p.codes[at.which] + block * 16 + 4 * at.quarter) = bad ? 0u : codes;
  if (at.quarter == 0) p.scales[at.which][block] = bad ? kC4Bad : static_cast<uint8_t>(e + 127);
}

template <typename T>
__global__ void __launch_bounds__(256) cache4_read_kernel(const Cache4Params p) {
  const int lane = static_cast<int>(threadIdx.x) & 63, units = 2 * p.kv_heads * p.blocks * 4, waves = (units + 63) / 64;
  const int64_t index = static_cast<int64_t>(blockIdx.x) * 4 + __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x >> 6));
  const int t = static_cast<int>(index / waves);
  if (t >= p.tokens) return;
  const int u = static_cast<int>(index - static_cast<int64_t>(t) * waves) * 64 + lane;
  const int64_t row = c4_row(p, t, lane);
  if (u >= units) return;
  const C4Unit at(p, u);
  const int ch = at.channel();
  if (ch >= p.dim) return;
  float v[8] = {};
  if (row >= 0) {
    const int64_t block = (at.head * static_cast<int64_t>(p.rows) + row) * p.blocks + at.block;
    const uint32_t scale = p.scales[at.which][block];
    c4_f32(*reinterpret_cast<const uint32_t*>(p.codes[at.which] + block * 16 + 4 * at.quarter), c4_scale(scale), v);
    if (scale > kC4Most) {
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = NAN;
    }
  }
  T* y = static_cast<T*>(p.y[at.which]) + static_cast<int64_t>(t) * p.st[at.which][0] + at.head * p.st[at.which][1] + ch;
  constexpr int E = 16 / static_cast<int>(sizeof(T));
#pragma unroll
  for (int j = 0; j < 8; j += E) rot_store<T>(y + j, v + j);
}

// ---- attention of few rows ---------------------------------------------------------------------
//
// A sequence's rows r = t G + g (packed_attention_kernels.h), 16 at a time, over one part of its keys. The four waves of
// a workgroup walk over the part's chunks of 64 keys in turn, each by itself, and join their sums in LDS: no barrier in
// the loop, and every wave has its own loads under way.
//
// Products of 16 x 16 x 32. S^T = K q^T: a lane holds one key and a quarter of the channels as they come from memory, 4 to
// 16 bytes, which become bf16 in registers (exactly, scale included), so keys touch no LDS; q's channels are dealt out to
// the lanes in that order. A lane then owns one row and 4 keys of each 16, whose weights are the B operand of the
// second product as they are. Its A operand, values along the keys, needs a transpose: 32 rows of bf16 in the wave's LDS
// with swizzled 16-byte pieces, read back by transposing reads.
//
// bf16 queries: the weights as two bf16 numbers (with one, results were 1.38 times as far off as the exact ones rounded,
// and the loads bound these calls). f32: q and the weights as three.

template <typename T>
constexpr int kC4QTerms = sizeof(T) == 2 ? 1 : 3;
template <typename T>
constexpr int kC4PTerms = sizeof(T) == 2 ? 2 : 3;
constexpr int kC4Rows = 16;

// x as N bf16 numbers that add up to it, 8 at a time.
template <int N>
__device__ __forceinline__ void c4_terms(at_f8 x, at_bf8 (&to)[N]) {
#pragma unroll
  for (int n = 0; n < N; ++n) {
    to[n] = __builtin_convertvector(x, at_bf8);
    if (n + 1 < N) x -= __builtin_convertvector(to[n], at_f8);
  }
}

__device__ __forceinline__ float c4_max_groups(float x) {  // over the lanes of equal lane % 16
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return at_max_halves(fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1])));
}
__device__ __forceinline__ float c4_sum_groups(float x) {
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return at_sum_halves(__uint_as_float(r[0]) + __uint_as_float(r[1]));
}

typedef uint32_t c4_u2 __attribute__((ext_vector_type(2)));
typedef uint32_t c4_u3 __attribute__((ext_vector_type(3)));
typedef uint32_t c4_u4 __attribute__((ext_vector_type(4)));

// A lane's share of 16 rows of the cache: a quarter of one row's channels.
template <int DT>
struct C4Rows {
  static constexpr int N = DT / 32, B = DT / 32;  // dwords of a share, blocks of a row
  uint32_t codes[N];
  uint32_t scale[DT == 96 ? 2 : 1];
  // Row 16 j + col of a chunk, whose codes and scales the two buffers hold: zeros behind its last row.
  __device__ __forceinline__ void load(__amdgpu_buffer_rsrc_t c, __amdgpu_buffer_rsrc_t s, int j, int col, int grp) {
    const int at = col * (DT / 2) + grp * (DT / 8), first = 16 * j * (DT / 2);
    if constexpr (N == 4) {
      const c4_u4 x = __builtin_amdgcn_raw_buffer_load_b128(c, at + first, 0, 0);
      codes[0] = x[0], codes[1] = x[1], codes[2] = x[2], codes[3] = x[3];
    } else if constexpr (N == 3) {
      const c4_u3 x = __builtin_amdgcn_raw_buffer_load_b96(c, at + first, 0, 0);
      codes[0] = x[0], codes[1] = x[1], codes[2] = x[2];
    } else if constexpr (N == 2) {
      const c4_u2 x = __builtin_amdgcn_raw_buffer_load_b64(c, at + first, 0, 0);
      codes[0] = x[0], codes[1] = x[1];
    } else {
      codes[0] = __builtin_amdgcn_raw_buffer_load_b32(c, at + first, 0, 0);
    }
    const int row = col * B + 16 * j * B;
    if constexpr (DT == 96) {  // 24 channels, of one block or two
      scale[0] = __builtin_amdgcn_raw_buffer_load_b8(s, row + 24 * grp / 32, 0, 0);
      scale[1] = __builtin_amdgcn_raw_buffer_load_b8(s, row + (24 * grp + 16) / 32, 0, 0);
    } else {
      scale[0] = __builtin_amdgcn_raw_buffer_load_b8(s, row + grp * (DT / 4) / 32, 0, 0);
    }
  }
  __device__ __forceinline__ uint32_t scale_of(int e, int grp) const {  // of dword e, channels grp DT / 4 + 8 e ..
    if constexpr (DT == 96) return e == 0 || (e == 1 && grp != 1) ? scale[0] : scale[1];
    else return scale[0];
  }
  __device__ __forceinline__ at_bf8 bf16(int e, int grp) const { return c4_bf16(codes[e], c4_scale(scale_of(e, grp))); }
  __device__ __forceinline__ bool bad() const {
    bool b = scale[0] > kC4Most;
    if constexpr (DT == 96) b = b || scale[1] > kC4Most;
    return b;
  }
};

// What bounds it: the loads, and the vector work beside them: 64 tokens over caches of 129 to 8,000 keys, 32 heads to 8 of
// 128 channels, 135 MB, 40 us (3.4 TB/s) with half of the vector units' time; with addresses formed and rows clamped for
// each load, and transposing reads that met on half of the banks, 43. Parts of 16 chunks: 8 45 us, 32 41.
template <typename T, int DT, bool SHAPED>
__global__ void __launch_bounds__(256, sizeof(T) == 2 ? 3 : 2) cache4_attention_kernel(const PackParams p) {
  constexpr int DP = DT == 96 ? 128 : DT, CPR = DP / 8;  // channels and 16-byte pieces of a row in LDS
  constexpr int N = DT / 32, MT = DT / 16, QT = kC4QTerms<T>, PT = kC4PTerms<T>;
  __shared__ __align__(16) unsigned char area[4][64 * DP];  // a wave's 32 rows of values, later its sums
  __shared__ float2 ml[4][kC4Rows];
  const int lane = static_cast<int>(threadIdx.x) & 63, wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x >> 6));
  const int grp = lane >> 4, col = lane & 15;
  // parts slowest, sequences, key heads: workgroups of parts that a sequence does not have come last
  const int b = static_cast<int>(blockIdx.x), cell = b / p.kv_heads, kv_head = b - cell * p.kv_heads;
  const int part = cell / (p.sequences + 1), seq = cell - part * (p.sequences + 1);
  T* out = static_cast<T*>(p.out);
  auto bound = [&](int s) { return min(max(p.q_offsets[s], 0), p.q_rows); };
  if (seq == p.sequences) {  // rows outside every sequence
    if (part != 0) return;
    const int before = bound(0), behind = bound(p.sequences), count = (before + p.q_rows - behind) * p.group, pieces = p.dim / 8;
    for (int64_t i = threadIdx.x; i < static_cast<int64_t>(count) * pieces; i += 256) {
      const int r = static_cast<int>(i / pieces), x = r / p.group, tok = x < before ? x : x - before + behind, h = kv_head * p.group + r - x * p.group;
      const int piece = static_cast<int>(i - static_cast<int64_t>(r) * pieces);
      T* to = out + tok * p.st[kPkO][0] + h * p.st[kPkO][1] + 8 * piece;
#pragma unroll
      for (int j = 0; j < 8; ++j) to[j] = T{};
      if (p.splits > 1 && piece == 0) p.part_n[static_cast<int64_t>(tok) * p.heads + h] = 1;
    }
    return;
  }
  const int q_first = bound(seq), n = bound(seq + 1) - q_first;
  if (n <= 0) return;
  const PkRange keys(p, seq);
  const int m = keys.count, shift = m - n, prefix = SHAPED && p.prefix != nullptr ? p.prefix[seq] : 0;
  auto seen = [&](int t) { return SHAPED ? pk_hi(p, t + shift, prefix, m) : p.causal ? max(t + shift + 1, 0) : m; };
  auto from = [&](int t) { return SHAPED ? pk_lo(p, t + shift) : 0; };
  // the chunks that some query sees, in parts of p.part, or more where that makes more than p.splits
  const int first = from(0) / kPkChunk, chunks = max((seen(n - 1) + kPkChunk - 1) / kPkChunk - first, 0);
  const int per = max(p.part, (chunks + p.splits - 1) / p.splits), parts = max((chunks + per - 1) / per, 1);
  if (part >= parts) return;
  const int c0 = first + part * per, c1 = min(first + chunks, c0 + per);
  const int64_t head_rows = static_cast<int64_t>(kv_head) * p.k_rows + keys.first;
  const uint8_t* kc = static_cast<const uint8_t*>(p.k) + head_rows * (DT / 2);
  const uint8_t* vc = static_cast<const uint8_t*>(p.v) + head_rows * (DT / 2);
  const uint8_t* ks = p.k_scales + head_rows * (DT / 32);
  const uint8_t* vs = p.v_scales + head_rows * (DT / 32);
  unsigned char* const mine = area[wave];
  // Piece c of row r lies at c ^ swizzle(r): 16 rows of one piece (the writes), and 8 rows of two neighbouring ones (half
  // a wave's transposing read), fall on 256 bytes of banks. Rows 16 apart have the same.
  auto swizzle = [](int r) { return (r / (16 / CPR) % (CPR / 2)) * 2 | (r >> 3 & 1); };
  // lane 4 j + a of a group reads key 4 grp + j, channels 4 a .. of 16
  const int key = 4 * grp + (col >> 2), quad = col & 3;
  const uint32_t read_at = key * (2 * DP) + (((quad >> 1) ^ swizzle(key)) << 4) + 8 * (quad & 1), write_at = col * (2 * DP);

  for (int r0 = 0; r0 < n * p.group; r0 += kC4Rows) {
    const int r = r0 + col, rc = min(r, n * p.group - 1), tok = rc / p.group, g = rc - tok * p.group, head = kv_head * p.group + g;
    const bool valid = r < n * p.group;
    const int lim = valid ? seen(tok) : 0, lo = from(tok), span = max(lim - lo, 0);
    const int t0 = r0 / p.group, t1 = (min(r0 + kC4Rows, n * p.group) - 1) / p.group;
    const int tile_end = seen(t1), tile_first = from(t0), full = r0 + kC4Rows <= n * p.group ? seen(t0) : 0, full_first = from(t1);
    at_bf8 q[N][QT];
#pragma unroll
    for (int e = 0; e < N; ++e) {
      const int ch = grp * (DT / 4) + 8 * e;
      float x[8] = {};
      if (valid && ch < p.dim) {
        const T* row = static_cast<const T*>(p.q) + (q_first + tok) * p.st[kPkQ][0] + head * p.st[kPkQ][1] + ch;
        constexpr int E = 16 / static_cast<int>(sizeof(T));
#pragma unroll
        for (int j = 0; j < 8; j += E) rot_load<T>(x + j, row + j);
      }
      c4_terms(at_f8{x[0], x[1], x[2], x[3], x[4], x[5], x[6], x[7]}, q[e]);
    }
    float slope = 0.0f;
    if (SHAPED && p.slopes != nullptr) slope = p.slopes[head] * -1.44269504f;
    const int place = tok + shift;
    float top = 0.0f, l = 0.0f;  // the running reference score; the sum over the lane's keys
    bool fresh = true, sick = false;
    at_f4 o[MT];  // channels 16 i + 4 grp .. of the lane's row
#pragma unroll
    for (int i = 0; i < MT; ++i) o[i] = at_f4{0.0f, 0.0f, 0.0f, 0.0f};

    C4Rows<DT> kr[4], vr[4];
    // A chunk is two buffers, whose addresses are the wave's: a lane adds a constant, and rows behind the last key need no
    // test of their own.
    auto load = [&](C4Rows<DT>(&x)[4], const uint8_t* codes, const uint8_t* scales, int c) {
      const int rows = __builtin_amdgcn_readfirstlane(min(m - c * kPkChunk, kPkChunk));
      const __amdgpu_buffer_rsrc_t cb = pk_buffer(codes + static_cast<int64_t>(c) * (kPkChunk * (DT / 2)), rows * (DT / 2));
      const __amdgpu_buffer_rsrc_t sb = pk_buffer(scales + static_cast<int64_t>(c) * (kPkChunk * (DT / 32)), rows * (DT / 32));
#pragma unroll
      for (int j = 0; j < 4; ++j) x[j].load(cb, sb, j, col, grp);
    };
    auto load_keys = [&](int c) { load(kr, kc, ks, c); };
    auto load_values = [&](int c) { load(vr, vc, vs, c); };
    // chunks that the tile's rows see
    const int ca = max(c0, tile_first / kPkChunk), cz = min(c1, (tile_end + kPkChunk - 1) / kPkChunk);
    int c = ca + wave;
    if (c < cz) {
      load_keys(c);
      load_values(c);
    }
    for (; c < cz; c += 4) {
      const int k0 = c * kPkChunk;
      at_f4 s[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        s[j] = at_f4{0.0f, 0.0f, 0.0f, 0.0f};
        const bool spoilt = __any(kr[j].bad());
#pragma unroll
        for (int e = 0; e < N; ++e) {
          at_bf8 a = kr[j].bf16(e, grp);
          if (spoilt && kr[j].scale_of(e, grp) > kC4Most) a[0] = static_cast<__bf16>(NAN);
#pragma unroll
          for (int t = QT - 1; t >= 0; --t) s[j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, q[e][t], s[j], 0, 0, 0);
        }
        if (j % 2 == 1) __builtin_amdgcn_sched_barrier(0);  // left to itself the compiler converts everything first: 230 registers
      }
      if (c + 4 < cz) load_keys(c + 4);
      if (SHAPED && p.cap2 != 0.0f) {
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
          for (int i = 0; i < 4; ++i) s[j][i] = fmaf(pk_bent<T>(p, s[j][i]), p.cap2, -top);
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
          for (int i = 0; i < 4; ++i) s[j][i] = fmaf(s[j][i], p.scale2, -top);
      }
      if (SHAPED && p.slopes != nullptr) {
        const float ahead = static_cast<float>(k0 + 4 * grp - place);  // (as integers: places from 2^24 on are not all floats)
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
          for (int i = 0; i < 4; ++i) s[j][i] = fmaf(slope, fabsf(ahead + static_cast<float>(16 * j + i)), s[j][i]);
      }
      if (k0 + kPkChunk > full || (SHAPED && k0 < full_first)) {
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            s[j][i] = static_cast<uint32_t>(k0 + 16 * j + 4 * grp + i - lo) < static_cast<uint32_t>(span) ? s[j][i] : -INFINITY;
      }
      float bm = -INFINITY;
#pragma unroll
      for (int j = 0; j < 4; ++j) bm = fmaxf(bm, fmaxf(fmaxf(s[j][0], s[j][1]), fmaxf(s[j][2], s[j][3])));
      if (__any(bm > kAtLazy || (fresh && bm != -INFINITY))) {
        bm = c4_max_groups(bm);
        const bool move = bm > kAtLazy || (fresh && bm != -INFINITY);
        const float d = move ? bm : 0.0f, alpha = !move ? 1.0f : fresh ? 0.0f : at_exp2(-d);
        top += d;
        l *= alpha;
        fresh = fresh && !move;
#pragma unroll
        for (int j = 0; j < 4; ++j) s[j] -= d;
#pragma unroll
        for (int i = 0; i < MT; ++i) o[i] *= alpha;
      }
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          s[j][i] = at_exp2(s[j][i]);
          l += s[j][i];
        }
#pragma unroll
      for (int h = 0; h < 2; ++h) {
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const C4Rows<DT>& x = vr[2 * h + j];
          const bool spoilt = __any(x.bad());
          sick = sick || spoilt;
#pragma unroll
          for (int e = 0; e < N; ++e) {
            uint4 y = __builtin_bit_cast(uint4, x.bf16(e, grp));
            if (spoilt && x.scale_of(e, grp) > kC4Most) y = uint4{0u, 0u, 0u, 0u};  // its rows get it in the end
            *reinterpret_cast<uint4*>(mine + (write_at + (((grp * N + e) ^ swizzle(col)) << 4)) + 16 * j * (2 * DP)) = y;
          }
          __builtin_amdgcn_sched_barrier(0);
        }
        if (h == 1 && c + 4 < cz) load_values(c + 4);
        at_bf8 w[PT];
        c4_terms(at_f8{s[2 * h][0], s[2 * h][1], s[2 * h][2], s[2 * h][3], s[2 * h + 1][0], s[2 * h + 1][1], s[2 * h + 1][2], s[2 * h + 1][3]}, w);
        pk_wave_sync();
#pragma unroll
        for (int i = 0; i < MT; ++i) {
          const PkLds at = (PkLds)(mine) + (read_at ^ (i << 5));
          const at_bf8 a = at_bf8_of(pk_read_tr(at), pk_read_tr(at + 16 * (2 * DP)));
#pragma unroll
          for (int t = PT - 1; t >= 0; --t) o[i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, w[t], o[i], 0, 0, 0);
          if (i % 4 == 3) __builtin_amdgcn_sched_barrier(0);
        }
        pk_wave_sync();
      }
    }
    if (sick) {  // blocks of values that are not finite: NaN for the rows that see them
      for (c = ca + wave; c < cz; c += 4)
        for (int j = c * kPkChunk; j < min((c + 1) * kPkChunk, m); ++j)
#pragma unroll
          for (int i = 0; i < MT; ++i)
            if (vs[static_cast<int64_t>(j) * (DT / 32) + i / 2] > kC4Most && j >= lo && j < lim) o[i] += at_f4{NAN, NAN, NAN, NAN};
    }
    l = c4_sum_groups(l);
    if (grp == 0) ml[wave][col] = float2{top, l};
#pragma unroll
    for (int i = 0; i < MT; ++i) *reinterpret_cast<at_f4*>(mine + col * (4 * DP) + (((4 * i + grp) ^ (col & (DP / 4 - 1))) << 4)) = o[i];
    __syncthreads();
    constexpr int C = DT / 4;
    for (int i = threadIdx.x; i < kC4Rows * C; i += 256) {
      const int x = i / C, ch = 4 * (i - x * C), row = r0 + x;
      if (row >= n * p.group || ch >= p.dim) continue;
      float best = -INFINITY, sum = 0.0f;
#pragma unroll
      for (int w = 0; w < 4; ++w)
        if (ml[w][x].y != 0.0f) best = fmaxf(best, ml[w][x].x);
      at_f4 a = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int w = 0; w < 4; ++w)
        if (ml[w][x].y != 0.0f) {
          const float f = at_exp2(ml[w][x].x - best);
          sum += ml[w][x].y * f;
          a += *reinterpret_cast<const at_f4*>(area[w] + x * (4 * DP) + (((ch >> 2) ^ (x & (DP / 4 - 1))) << 4)) * f;
        }
      const int tk = row / p.group, hd = kv_head * p.group + row - tk * p.group;
      const int64_t stat = static_cast<int64_t>(q_first + tk) * p.heads + hd;
      if (parts == 1) {
        pk_put4(out + (q_first + tk) * p.st[kPkO][0] + hd * p.st[kPkO][1] + ch, sum == 0.0f ? a : a * (1.0f / sum));
      } else {
        const int64_t at = static_cast<int64_t>(part) * p.q_rows * p.heads + stat;
        *reinterpret_cast<at_f4*>(p.part_o + at * p.dim + ch) = a;
        if (ch == 0) *reinterpret_cast<float2*>(p.part_ml + at * 2) = float2{sum == 0.0f ? 0.0f : best, sum};
      }
      if (p.splits > 1 && part == 0 && ch == 0) p.part_n[stat] = parts;
    }
    __syncthreads();
  }
}

}  // namespace msda
