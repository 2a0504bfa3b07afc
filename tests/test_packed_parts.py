"""How the packed attention's forward shares a tile's keys between workgroups (csrc/packed_attention_parts.h), on the CPU:
the header is compiled by g++ into a program that walks over random calls, traps on overflow, and counts the kinds of
calls that it met."""

from __future__ import annotations

import os
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

PROGRAM = r"""
#include "packed_attention_parts.h"

#include <cmath>
#include <cstdio>
#include <random>

using namespace msda;

int main() {
  std::mt19937_64 rng(7);
  auto upto = [&](int64_t lo, int64_t hi) {  // its logarithm uniform
    const double u = static_cast<double>(rng() >> 11) * 0x1p-53;
    return std::min(hi, std::max(lo, static_cast<int64_t>(std::llround(lo * std::pow(static_cast<double>(hi) / lo, u)))));
  };
  long split = 0, growing = 0, blind = 0, longer = 0;
  for (int i = 0; i < 200000; ++i) {
    const bool big = i % 4 == 0, prompt = i % 4 == 1;  // prompt: as many keys as queries, few and alike sequences
    const int group = static_cast<int>(upto(1, prompt ? 4 : 64)), kv_heads = static_cast<int>(upto(1, 64)), sequences = static_cast<int>(upto(1, prompt ? 4 : 2000));
    const int64_t most_rows = big ? (int64_t{1} << 31) / group - 128 * (sequences + 4) : 20000;
    if (most_rows < 2) continue;
    const int q_rows = static_cast<int>(upto(1, most_rows)), k_rows = prompt ? q_rows : static_cast<int>(upto(1, big ? (int64_t{1} << 31) - 128 * (sequences + 4) : 100000));
    const PackShape s{i % 2, sequences, q_rows, k_rows, group * kv_heads, kv_heads, 64};
    const PackSplit at = pk_split(s);
    if (at.most == 1) continue;
    ++split;
    if (at.most < 3 || at.most > kPkMostParts || at.part < 2) return std::printf("split %d %d\n", at.most, at.part), 1;
    for (int j = 0; j < 8; ++j) {  // any lengths of sequences in such a call
      const int n = static_cast<int>(prompt && j < 4 ? std::max(q_rows / sequences - 100 * j, 1) : upto(1, q_rows));
      const int m = prompt && j < 3 ? n : static_cast<int>(j == 0 ? k_rows : upto(1, k_rows));
      const bool causal = j % 4 != 3;
      const PkParts parts(at.most, at.part, causal, group, n, m);
      const int tiles = static_cast<int>((static_cast<int64_t>(n) * group + kPkTile - 1) / kPkTile);
      auto chunks = [&](int tile) {  // that the tile's last row sees
        const int64_t row = std::min<int64_t>(static_cast<int64_t>(tile + 1) * kPkTile, static_cast<int64_t>(n) * group) - 1;
        const int64_t seen = causal ? std::min<int64_t>(std::max<int64_t>(row / group + m - n + 1, 0), m) : m;
        return static_cast<int>((seen + kPkChunk - 1) / kPkChunk);
      };
      if (tiles <= 600) {
        int sum = 0;
        for (int t = 0; t < tiles; ++t) {
          const int of = parts.of(t);
          if (parts.before(t) != sum) return std::printf("before(%d) %d, sum %d; %d %d\n", t, parts.before(t), sum, n, m), 1;
          if (of < 1 || of > at.most) return std::printf("of(%d) %d of %d\n", t, of, at.most), 1;
          sum += of;
        }
        if (parts.before(tiles) != sum) return std::printf("before(%d) %d, sum %d\n", tiles, parts.before(tiles), sum), 1;
      } else {
        for (int x = 0; x < 50; ++x) {
          const int t = x == 0 ? tiles - 1 : static_cast<int>(upto(1, tiles)) - 1, of = parts.of(t);
          if (parts.before(t + 1) - parts.before(t) != of || of < 1 || of > at.most) return std::printf("of(%d) %d of %d\n", t, of, at.most), 1;
        }
        if (parts.before(0) != 0) return 1;
      }
      // the last tile's parts, from which the host's room for two more follows
      const int last = chunks(tiles - 1), room = at.most - 2, part = std::max(at.part, (last + room - 1) / room);
      if ((parts.of(tiles - 1) - 1) * static_cast<int64_t>(part) >= last + 2) return std::printf("%d parts of %d chunks, %d each\n", parts.of(tiles - 1), last, part), 1;
      growing += parts.of(tiles - 1) > parts.first;
      blind += parts.from > 0;
      longer += part > at.part;
    }
  }
  std::printf("%ld %ld %ld %ld\n", split, growing, blind, longer);
  return 0;
}
"""


def test_parts_of_random_calls(tmp_path):
    source, program = tmp_path / "parts.cpp", tmp_path / "parts"
    source.write_text(PROGRAM)
    include = [f for d in ("rf-detr-jax_amd/csrc", "include") for f in ("-I", os.path.join(ROOT, d))]
    subprocess.run(["g++", "-std=c++17", "-O2", "-ftrapv", "-Wall", "-Werror", *include, str(source), "-o", str(program)], check=True)
    done = subprocess.run([str(program)], capture_output=True, text=True, timeout=100)
    assert done.returncode == 0, done.stdout
    split, growing, blind, longer = map(int, done.stdout.split())
    assert min(split, growing, blind, longer) > 1000, done.stdout


@pytest.mark.parametrize("change", ["x * first + q", "step = (part * group + 1) / 2", "room = splits - 2"])
def test_a_planted_mistake_is_found(tmp_path, change):
    """The program on a header with one mistake in it."""
    mistake = {"x * first + q": "x * first + 1 + q", "step = (part * group + 1) / 2": "step = (part * group + 1) / 4 + 1", "room = splits - 2": "room = splits"}
    with open(os.path.join(ROOT, "rf-detr-jax_amd/csrc/packed_attention_parts.h")) as f:
        header = f.read()
    assert header.count(change) == 1
    (tmp_path / "packed_attention_parts.h").write_text(header.replace(change, mistake[change]))
    source, program = tmp_path / "parts.cpp", tmp_path / "parts"
    source.write_text(PROGRAM)
    subprocess.run(["g++", "-std=c++17", "-O2", "-I", str(tmp_path), "-I", os.path.join(ROOT, "include"), str(source), "-o", str(program)], check=True)
    assert subprocess.run([str(program)], capture_output=True, timeout=100).returncode != 0
