// How a call of llmk_lora_add is cut into launches and blocks, by its sizes alone: host arithmetic only (not
// exported). lora.hip has the kernels and what they measured.
#pragma once
#include <math.h>
#include <stddef.h>

namespace llmk {
namespace lora {

constexpr int kParts = 8, kMaxRank = 256;
constexpr int kWindow = 256;  // sequences whose tiles are found together
constexpr int kRows = 16;     // of a tile
constexpr int kChunk = 256;   // of in_features that a wave takes at a time
constexpr int kWaves = 8;     // of a block of k_lora_whole

// Blocks that k_lora_shrink is given if it has as many. 512: 3 prompts of 456 rows and rank 128 on 8192 -> 11008|11008
// take 100 us and not 92, of rank 64 on 4096 -> 4096|1024|1024 42.7 and 41; the other cases as long.
constexpr int kFill = 1024;

constexpr int kMostBlocks = (1 << 24) - 1;  // of 256 threads, which a launch counts in 32 bits

inline int over(long long a, long long b) { return (int)((a + b - 1) / b); }

inline bool within_limits(int n_rows, int n_seqs, int max_rank, int in) {
  return max_rank <= kMaxRank && n_rows <= (1 << 20) && n_seqs <= (1 << 20) && in <= (1 << 24);
}

// What a call takes of the chip and the workspace.
struct Shape {
  int groups, windows, slots, splits;
  int at_once, turns;  // products of 16 ranks that a block of k_lora_shrink computes at a time, blocks that take turns
};
inline Shape shape_of(int n_rows, int n_seqs, int n_adapters, int in, int products) {
  Shape s;
  s.groups = n_seqs < kWindow ? n_seqs : kWindow;
  if (n_adapters < s.groups) s.groups = n_adapters;
  s.windows = (n_seqs + kWindow - 1) / kWindow;
  s.slots = n_rows / kRows + s.windows * (s.groups + 1);
  // one at a time where tiles are few: one row of rank 128 on 4096 -> 11008|11008 takes 13.5 us and not 14.2 with
  // two, 32 rows of rank 16 on 8192 -> 4096|1024|1024 10.6 and not 11.9 with three; but 256 rows of 100 adapters of
  // up to 64 29.2 and not 28.7, 3 prompts of 456 rows and rank 128 110 and not 89
  s.at_once = products == 1 || s.slots * products <= 256 ? 1 : products == 3 ? 3 : 2;
  // blocks for the products first, as long as kFill are not there, then for parts of in_features, whose sums every
  // block of k_lora_expand has to add up
  const int passes = (products + s.at_once - 1) / s.at_once, most = (in + 4 * kChunk - 1) / (4 * kChunk);
  const int want = (kFill + s.slots - 1) / s.slots;
  s.turns = want < passes ? want : passes;
  s.splits = (kFill + s.slots * s.turns - 1) / (s.slots * s.turns);
  if (s.splits > most) s.splits = most;
  if (s.splits > 8) s.splits = 8;  // what k_lora_expand adds up
  const int each = (most + s.splits - 1) / s.splits;
  s.splits = (most + each - 1) / each;  // none idle at the end
  return s;
}

// How many tiles there will be about if sequences choose among the adapters evenly, and if all choose another.
struct Tiles {
  int likely, many;
};
inline Tiles tiles_of(int n_rows, int n_seqs, int n_adapters, int windows, int groups) {
  const double n = n_seqs < kWindow ? n_seqs : kWindow, rows = n_rows / (double)kRows, most = (double)windows * groups;
  // adapters that are asked for, of those there are; without a difference of numbers near 1, and a whole number is one
  const double some = (double)windows * n_adapters * -expm1(n * log1p(-1.0 / n_adapters));
  return {(int)(fmax(some, rows + 0.5 * (some - 1)) + 1e-6), (int)ceil(fmax(most, rows + 0.75 * (most - 1)))};
}

// The launches: both products in one, or in two.
struct Launches {
  bool one;
  int tiles;      // one: 16 columns each, of a wave
  bool together;  // one: a tile's blocks share an XCD
  int blocks;     // one: of a tile
  int per_block;  // two: tiles of a block of the second
  int steps;      // of 32 ranks, that its kernels are made for: 1, 2, 4 or 8
  int columns;    // of a block of the second
  size_t grid, grid2;  // one: blocks; two: of the first and of the second
};

// part_ends: ascending, of n_parts parts; s: shape_of these sizes. One launch where a block's own h costs it little, 32
// ranks at most and few enough numbers of A and x, and where its blocks are expected to run at once: one a CU, 32 an
// XCD. Columns a block: 256, 512 or 1024, the fewest with which they do. 300 rows of one adapter of rank 16 on 1024 ->
// 6144 take 7.9 us and 9.0 in two launches (12.0 if a third of an XCD's blocks waits for the others), on 11008|11008
// 20.0 so and 15.9. 16 ranks and 2048 columns of one sequence take 5.9 us with 4096 in_features and 7.8 with 8192,
// where two launches take 8.1; 16 sequences' on 1000 columns 9.4 and 10.8, but one sequence of 16 rows 9.9 and 8.9, and
// 32 sequences of 4 adapters 11.0 and 9.9: there x counts as much as A. At 32 ranks 8 sequences on 4096 ->
// 4096|1024|1024 take 9.5 and 11.3, 4 of 16 rows on 8192|8192, 1024 columns a block, 12.4 and 10.6. A launch more is 2
// us of the host's time, too. The columns are chosen for many tiles, as too few of them cost more: 48 sequences of up
// to 5 rows, 16 adapters, 4096 -> 4096|1024|1024, 11.2 us with 1024 and 14.6 with 512, of which a third has to wait on
// some XCDs.
inline Launches launches_of(const Shape& s, int n_rows, int n_seqs, int n_adapters, int max_rank, int in,
                            const int* part_ends, int n_parts) {
  Launches l{};
  l.steps = max_rank <= 32 ? 1 : max_rank <= 64 ? 2 : max_rank <= 128 ? 4 : 8;
  l.columns = l.steps <= 4 ? 512 : 256;
  const int per_part = (max_rank + 15) / 16;
  const auto blocks_of = [&](int columns) {
    int blocks = 0;
    for (int p = 0; p < n_parts; ++p) blocks += over(part_ends[p] - (p ? part_ends[p - 1] : 0), columns);
    return blocks;
  };
  const Tiles used = tiles_of(n_rows, n_seqs, n_adapters, s.windows, s.groups);
  const auto fits = [&](long long n) { return l.together ? (n + 7) / 8 * l.blocks <= 32 : n * l.blocks <= 256; };
  for (l.tiles = 2;; l.tiles *= 2) {
    l.blocks = blocks_of(16 * kWaves * l.tiles);
    l.together = s.slots >= 8 || l.blocks <= 32;
    if (l.tiles == 8 || fits(used.many)) break;
  }
  const size_t most = per_part == 1 && n_rows < 8 * s.groups ? 16384 : l.tiles == 8 ? 10240 : 12288;
  l.one = fits(used.likely) && l.steps == 1 && (per_part + 1) * (size_t)in <= most;
  l.grid = l.one ? (size_t)(l.together ? (s.slots + 7) / 8 * 8 : s.slots) * l.blocks
                 : (size_t)s.splits * s.slots * s.turns;
  // as many tiles a block as leave 2048 blocks, or 512 past 32 ranks, where B is more than y: 2 prompts of 900 rows and
  // rank 64 on 8192|8192 columns take 32 us, and 40 with 2048
  const int chunks = blocks_of(l.columns);
  l.per_block = 1;
  while (l.per_block < 16 && (long long)s.slots * chunks / (2 * l.per_block) >= (l.steps == 1 ? 2048 : 512))
    l.per_block *= 2;
  while ((size_t)chunks * over(s.slots, l.per_block) > kMostBlocks) l.per_block *= 2;  // ends: chunks are 65535 at most
  l.grid2 = (size_t)chunks * over(s.slots, l.per_block);
  return l;
}

}  // namespace lora
}  // namespace llmk
