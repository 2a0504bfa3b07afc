// packed_attention_parts.h — how the forward of the packed attention shares a tile's keys between workgroups:
// the host's choice from the sums of lengths, and the numbers of parts that the device forms from the lengths.
// Plain constexpr C++, for both and for a test on the CPU.
#pragma once

#include <algorithm>
#include <cstdint>

#include "msda.h"

namespace msda {

constexpr int kPkWaves = 4;              // of a workgroup
constexpr int kPkTile = 32 * kPkWaves;   // own rows of a workgroup: 32 a wave
constexpr int kPkChunk = 64;             // streamed rows of a tile
constexpr int kPkMostParts = 64;  // of a forward tile's keys

// One call's sizes.
struct PackShape {
  int dtype, sequences, q_rows, k_rows, heads, kv_heads, head_dim;
};

// The forward's split of the keys over workgroups: how many at most share a tile of rows, and the chunks of 64 keys
// that make one worth it. The lengths are not known here, only their sums; a workgroup finds its tile's number
// of parts from the length (PkParts).
struct PackSplit {
  int most, part;
};

inline PackSplit pk_split(const PackShape& s) {
  const PackSplit none{1, 1 << 30};
  if (s.sequences == 0) return none;
  const int64_t rows = static_cast<int64_t>(s.q_rows) * (s.heads / s.kv_heads);
  const int64_t tiles = std::min<int64_t>(rows, rows / kPkTile + s.sequences) * s.kv_heads;
  const int64_t chunks = (s.k_rows / s.sequences + kPkChunk - 1) / kPkChunk;  // of an average sequence
  if (tiles == 0) return none;
  // The work in parts that even out over the CUs: in bf16 one to each of the two workgroups that a CU holds, in f32 8
  // to a CU. The chunks counted here are those of the keys' room, not of their lengths, so there may be fewer parts with
  // work than wanted (3 caches of 16,384 rows, 30,022 keys in them: 380 for 512). One sequence of 6,000 tokens, 8 heads, causal (376 tiles,
  // the last of 94 chunks), us a call: bf16, 128 channels 131 with a workgroup a tile, 107 in 512 parts, 114 in
  // 2048; f32, 64 channels 532, 432 and 360. (Batches whose tiles even out by themselves pay for it: 512 tiles of 16
  // chunks in f32 175 us for 145.)
  const bool bf = s.dtype == MSDA_DTYPE_BF16;
  const int64_t wanted = bf ? 512 : 2048, even = (tiles * chunks + wanted - 1) / wanted;
  // Few rows to a tile on average (new tokens over caches): a part's own cost is small against its keys, so a call of
  // any size is split, because the longest cache would set its time. Full tiles: a part writes and the join reads 128
  // rows of f32 sums, the time of about 6 chunks of keys at 128 channels in bf16; in f32 (300 keys, 32 channels) parts of
  // 2 chunks cost 41 us for 31. The choice is one for the whole batch: a chunk of 512 tokens (32 heads) among 63 single
  // ones over caches of up to 8,000 keys makes the average row count large, nothing is split, and the longest cache
  // does set the time: 238 us, where 64 single tokens take 121.
  const bool few = rows <= int64_t{32} * s.sequences;
  const int64_t part = few ? std::clamp<int64_t>(even, 2, 16) : std::max<int64_t>(even, bf ? 6 : 8);
  if (chunks <= part) return none;
  // An average sequence's parts, for full tiles twice those (a longer one's are longer)
  const int64_t most = std::min<int64_t>((few ? 1 : 2) * ((chunks + part - 1) / part), kPkMostParts - 2);
  return PackSplit{static_cast<int>(most) + 2, static_cast<int>(part)};  // (PkParts: room for two more)
}

// The split forward: how many workgroups share tile i of a sequence of n queries and m keys. At least `part` chunks
// of keys each (more where a long sequence would make more parts than `splits`); a causal sequence's
// tiles see 2 / G chunks more from one to the next, so every `step` tiles make one part more, from the first tile
// that sees a key on, and the parts of the first x tiles have a closed form. With c chunks seen by the last tile
// and the tile sizes' roundings it has fewer than 1 + (c + 2) / part parts, at most room + 2 = splits.
struct PkParts {
  int first, from, step;
  constexpr PkParts(int splits, int part, bool causal, int group, int n, int m) : first(1), from(0), step(1 << 30) {
    const int shift = m - n, most = (m + kPkChunk - 1) / kPkChunk, room = splits - 2;  // most: chunks that the last tile sees
    if (most > part * room) part = (most + room - 1) / room;
    int chunks = most;  // that the first tile with keys sees
    if (causal && n * group > kPkTile) {
      from = shift < 0 ? -shift * group / kPkTile : 0;
      step = (part * group + 1) / 2;
      const int token = (std::min((from + 1) * kPkTile, n * group) - 1) / group;
      chunks = (std::min(std::max(token + shift + 1, 0), m) + kPkChunk - 1) / kPkChunk;
    }
    first = std::max((chunks + part - 1) / part, 1);
  }
  constexpr int of(int tile) const { return tile - from < step ? first : first + (tile - from) / step; }
  constexpr int before(int x) const {
    const int y = std::max(x - from, 0);
    if (y <= step) return x * first;
    const int q = y / step;
    return x * first + q * (q - 1) / 2 * step + q * (y - q * step);
  }
};

}  // namespace msda
