// Attention over the 8-bit KV cache (layout: kv8.hpp): out = softmax_j(q . K_j / sqrt(head_dim))
// V_j over the positions j up to the row's own, for rows of any number a sequence.
//
// One pass with a running maximum m and sum l in 32 bits: of a step's scores s, in log2 units,
//   m' = max(m, s), l' = 2^(m - m') l + sum 2^(s - m'), O' = 2^(m - m') O + sum 2^(s - m') V,
// and O / l at the end, rounded once. Both products run on the matrix cores, transposed, so that a
// row of q (a column here) stays in its lanes from the scores to the weights. K and V become fp16
// and bf16 on the way, exactly: v_cvt_scalef32_pk takes a block's scale along, and 4 significant
// bits fit both. Weights enter as two bf16, whatever their size: single ones of 8 or 11 bits would
// be the largest error of the result, and fp16 would lose those below 2^-24 of the maximum, of
// which a long context has many. That doubles the second product.
//
// What bounds it. A decode step reads 2 n_kv_heads head_dim bytes a position and uses each 4 times
// for each query head of a group: HBM, and the matrix cores only because the vector units, with
// e4m3 to convert and weights to make, would be slower than it (256 sequences of up to 2048
// positions 1494 us there). 256 sequences 59 us for 283 MB, 43.6 at a large copy's 6.5 TB/s; 3 of
// up to 65001 positions 48.5 us for 242 MB (37.2). Prompts are bound by the vector and the matrix
// units one after the other: a weight takes about 7 vector instructions (scale and subtract,
// exponential, sum, split) and 3 products, and by the counters a SIMD has vector instructions at
// work for 71 thousand cycles and products for 41 of the 115 thousand that its two waves live. They
// meet at a barrier every step, so neither hides the other. 1507 rows behind 1494 positions, 32
// heads of 64 dims, 65 us, 427 TFLOP/s of the definition's two products.
//
// Two kernels: waves on their own for few columns (k_kv8_attention_few) and blocks that share K and
// V through LDS for many. In both the work is cut into equal shares across the ends of sequences,
// and a second launch joins what several workers have of one unit.
#include <math.h>

#include <type_traits>

#include "kv8.hpp"
#include "kv8_shared.hpp"

namespace llmk {
namespace {

using namespace kv8;

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

constexpr float kLog2e = 1.44269504088896341f;
// Below it a rounded maximum (in log2 units) is less than 2^6 short of the exact one, which neither
// weights nor sums mind; from there on exponents are made in two steps, and the largest weight is
// 1.
constexpr float kLargeScore = 1073741824.0f;
// A row's weights are relative to a maximum that gives way only to one larger by more than this (in
// log2 units): they reach 2^kSlack, and sums are seldom rescaled.
constexpr float kSlack = 8.0f;
// What a unit's beginning costs, in steps. With 0 / 1 / 2 / 4, us: 48 sequences of up to 5 rows
// 41.1 / 37.5 / 35.8 / 36.1, 1507 rows of one 68.2 / 68.5 / 67.5 / 72.0.
constexpr int kStart = 2;
// Sequences of up to this many columns go by waves, in tiles of 32, where no sequence of the call
// has more; us by waves and by blocks: 48 x 16 rows (64 columns) 58.5 and 67.5, 4 x 16 19.9 and
// 23.4, 48 x 24 rows (96 columns) 82.7 and 74.0. Beside longer ones, up to kMixedColumns: blocks
// run anyhow, and the waves' launch stands in front of theirs (20 x up to 100 rows, 46.7 us with 32
// and 56.7 with 64).
constexpr int kFewColumns = 64, kMixedColumns = 32;
// From here on blocks of 8 waves and 256 columns: 1507 rows at 64 dims 74.0 -> 69.5 us, 500 rows at
// 128 dims 60.0 -> 53.8, 5 x 500 rows at 8000 positions 234 -> 206. Below, tiles of 128 columns
// leave fewer waves without work (32 query heads on 8, us, both at 2000 positions: 250 rows 27.9
// and 29.3, 100 rows 21.7 and 25.4, 20 x up to 100 rows 46.0 and 54.2).
constexpr int kWideColumns = 1024;
// Workers of a launch: a wave for each SIMD (256 sequences, us: 512 waves 92.1, 768 69.7, 1024
// 59.9, 1280 77.0, 2048 62.0 with twice the parts to join), or as many blocks as give it two. Two
// waves where each finds a unit of 16 columns or more of them and tables are of up to kShortPages
// pages, so that units are many and their beginnings the most of it: 256 sequences of up to 180,
// 300, 600 and 1000 positions 18.4 -> 16.8, 22.9 -> 21.7, 28.8 -> 27.7 and 36.4 -> 36.6 us.
constexpr int kFewWorkers = 1024, kShortPages = 40;
template <int W>
constexpr int kManyWorkers = 2048 / W;
constexpr int kWorkers = 2048, kMostKvHeads = 512;  // at most
constexpr int kSlotColumns = 131072;                // of partial results in the workspace
// With tables of up to this many pages units stay whole, and nothing is joined. Us with units
// shared and whole, one sequence, 64 of them and one of 5 rows: 192 positions of 64 dims 8.7 and
// 7.4, 11.5 and 9.0, 10.9 and 10.4 (256: 9.5 and 9.6, 11.6 and 9.8, 11.3 and 13.5); 128 of 128 dims
// 9.5 and 8.7, 13.0 and 10.6, 12.0 and 12.1.
constexpr int whole_pages(int head_dim) { return head_dim == 64 ? 12 : 8; }

template <bool HIGH>
__device__ __forceinline__ uint32_t bf16_from_e4m3(uint32_t bytes, float scale) {
  return __builtin_bit_cast(uint32_t,
                            __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(bytes, scale, HIGH));
}

// Two weights as packed bf16: their first 8 bits, and what that leaves rounded to 8 more, so that a
// weight keeps 16 bits or nearly so at any size. In one way the first are cut off.
__device__ __forceinline__ void split_cut(float a, float b, uint32_t& hi, uint32_t& lo) {
  const uint32_t x = __builtin_bit_cast(uint32_t, a), y = __builtin_bit_cast(uint32_t, b);
  hi = __builtin_amdgcn_perm(y, x, 0x07060302);
  const float ra = a - __builtin_bit_cast(float, x & 0xFFFF0000u);
  const float rb = b - __builtin_bit_cast(float, y & 0xFFFF0000u);
  const bf16x2 r = {(__bf16)ra, (__bf16)rb};
  lo = __builtin_bit_cast(uint32_t, r);
}
// In the other they are rounded, and what is left is a product of the packed halves with (-1, 0) or
// (0, -1) added to the weight: exact, and 4 instructions where the first way takes 6. Units of few
// columns gain by it (48 sequences of up to 5 rows: 36.2 -> 35.3 us); those of many, whose matrix
// instructions run beside it, lose (1507 rows: 84.6 -> 86.2 us).
__device__ __forceinline__ void split_rounded(float a, float b, uint32_t& hi, uint32_t& lo) {
  const bf16x2 h = {(__bf16)a, (__bf16)b};
  // from registers: as an operand in the instruction, -1 in the low half is taken for the high one
  uint32_t first = 0x0000BF80u, second = 0xBF800000u;
  asm("" : "+s"(first), "+s"(second));
  const float ra =
      __builtin_amdgcn_fdot2_f32_bf16(h, __builtin_bit_cast(bf16x2, first), a, false);
  const float rb =
      __builtin_amdgcn_fdot2_f32_bf16(h, __builtin_bit_cast(bf16x2, second), b, false);
  const bf16x2 r = {(__bf16)ra, (__bf16)rb};
  hi = __builtin_bit_cast(uint32_t, h);
  lo = __builtin_bit_cast(uint32_t, r);
}

// A running sum of the steps' sums of weights that takes along what each addition lost. A worker
// may walk a unit of 10^5 positions by itself, and equal weights added pair by pair lose the same
// way each time: 2^-11 of the sum at 131072 positions, as much as the result's own rounding. So it
// is the 32 additions of a step at most that count, less than 2^-20. O has no such help: a
// position's value is one of 32 (16) in a sum that the matrix cores add twice, so it may be off by
// 2^-28 (2^-27) of itself for each position, where weights and values are all equal: past 2^-11.5
// there at 131072 positions, and 2^-18 with weights that differ.
struct Sum {
  float of, lost;
  __device__ __forceinline__ void add(float x) {
    const float y = x - lost, next = of + y;
    lost = (next - of) - y;
    of = next;
  }
  __device__ __forceinline__ void scale(float by) {
    of = of * by;
    lost = lost * by;
  }
};

struct AttentionArgs {
  Batch batch;
  const f16* q;
  const uint8_t* k_pool;
  const float* k_scale;
  const uint8_t* v_pool;
  const float* v_scale;
  f16* out;
  float* parts;  // [2 workers][columns of a tile][HD], NULL: no unit is shared
  float2* parts_ml;
  Shared* shared;  // [2 workers]
  int n_heads, n_kv_heads, group, workers, teams;  // teams: workers / n_kv_heads
  int least_columns, most_columns;  // of the sequences that a launch takes
};

// A sequence's rows in this call and what they see.
struct Seq {
  int row0, columns;  // columns: (row, query head of the group) pairs, row by row
  long long before;   // position of the first row
  long long limit;    // positions that exist
};
__device__ __forceinline__ Seq seq_of(const AttentionArgs& a, int s) {
  Seq q;
  int r0 = s, r1 = s + 1;
  if (a.batch.starts) {
    r0 = a.batch.starts[s];
    r1 = a.batch.starts[s + 1];
  }
  const int len = a.batch.lens[s];
  q.before = (long long)len - (r1 - r0);
  r0 = r0 < 0 ? 0 : r0;
  r1 = r1 > a.batch.n_rows ? a.batch.n_rows : r1;
  q.row0 = r0;
  q.columns = r1 > r0 ? (r1 - r0) * a.group : 0;
  // none of another launch's
  if (q.columns < a.least_columns || q.columns > a.most_columns) q.columns = 0;
  const long long table = (long long)a.batch.max_pages * kPage;
  q.limit = len < table ? len : table;
  return q;
}
// Positions that the row of a column sees.
__device__ __forceinline__ int seen(const AttentionArgs& a, const Seq& q, int column) {
  const long long n = q.before + column / a.group + 1;
  const long long m = n < q.limit ? n : q.limit;
  return m < 0 ? 0 : (int)m;
}
// Columns in front of the first that sees something.
__device__ __forceinline__ int blind_of(const AttentionArgs& a, const Seq& q) {
  const long long n = q.limit <= 0 ? q.columns : -q.before * a.group;
  return n <= 0 ? 0 : n < q.columns ? (int)n : q.columns;
}
// A step of units of C columns: 16 bytes of K and as many of V for each of a block's threads, or,
// of the 64 of a wave, for each of 4 times.
template <int HD, int C>
constexpr int kPages = (C > 128 ? 512 : 256) / HD;
template <int HD, int C>
constexpr int kStep = kPages<HD, C> * kPage;

// Steps of a tile: those of its last row; one for a tile that sees nothing, which writes zeros. A
// unit's share of the work is counted in ticks, its steps and kStart for its beginning.
template <int HD, int C>
__device__ __forceinline__ int tile_steps(const AttentionArgs& a, const Seq& q, int tile) {
  const int last = (tile + 1) * C < q.columns ? (tile + 1) * C - 1 : q.columns - 1;
  const int n = (seen(a, q, last) + kStep<HD, C> - 1) / kStep<HD, C>;
  return n > 0 ? n : 1;
}
// Values that are the same in every lane, as scalars.
__device__ __forceinline__ int same(int x) { return __builtin_amdgcn_readfirstlane(x); }
__device__ __forceinline__ long long same(long long x) {
  const uint32_t lo = __builtin_amdgcn_readfirstlane((int)(uint32_t)x);
  const uint32_t hi = __builtin_amdgcn_readfirstlane((int)(uint32_t)((uint64_t)x >> 32));
  return (long long)(((uint64_t)hi << 32) | lo);
}

__device__ __forceinline__ Seq same(Seq q) {
  q.row0 = same(q.row0);
  q.columns = same(q.columns);
  q.before = same(q.before);
  q.limit = same(q.limit);
  return q;
}

// How a launch's work is shared out. A kv head's units are the tiles of all sequences, one behind
// the other; its ticks are cut into as many equal shares as there are teams, and a team has a
// worker for each kv head. So the heads of a page, which lie beside one another in memory, are read
// at about the same time (256 sequences 63.1 -> 61.8 us). Worker t n_kv_heads + h is head h's of
// team t; workers are waves or blocks. Who finds a share depends on how many sequences and tiles
// there are: a wave's lanes for up to 256, else the block's threads.
struct Share {
  int team, head, teams;
  int seq, tile;         // that hold the beginning of the team's share, and
  int at;                // its place in them, in ticks
  Seq rows;              // the sequence's
  long long begin, end;  // among the ticks of a head
  long long each;        // of the first `more` teams one more
  int more;
  __device__ __forceinline__ long long begin_of(int team) const {
    return each * team + (team < more ? team : more);
  }
  __device__ __forceinline__ int team_at(long long tick) const {
    const long long wide = (each + 1) * more;
    return (int)(tick < wide ? divide(tick, each + 1) : more + divide(tick - wide, each));
  }
  static __device__ __forceinline__ long long divide(long long a, long long b) {  // b > 0
    return (uint64_t)(a | b) >> 32 ? a / b : (long long)((uint32_t)a / (uint32_t)b);
  }
  // all but the place of the beginning
  static __device__ __forceinline__ Share of(const AttentionArgs& a, long long total, int worker) {
    Share r = {};
    r.teams = a.teams;
    if (total < r.teams) r.teams = total > 0 ? (int)total : 1;
    r.each = divide(total, r.teams);
    r.more = (int)(total - r.each * r.teams);
    r.team = worker / a.n_kv_heads;
    r.head = worker % a.n_kv_heads;
    r.begin = r.team < r.teams ? r.begin_of(r.team) : total;
    r.end = r.team < r.teams ? r.begin_of(r.team + 1) : total;
    return r;
  }
};

// The sum of the lanes up to each, by lane moves: within 16 lanes, then the rows in front (their
// last lanes').
template <int CTRL, int ROWS = 0xF>  // 0 where there is no source lane, and in rows not named
__device__ __forceinline__ long long dpp_i64(long long v) {
  const uint32_t lo =
      __builtin_amdgcn_update_dpp(0, (int)(uint32_t)v, CTRL, ROWS, 0xF, ROWS == 0xF);
  const uint32_t hi = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)((uint64_t)v >> 32), CTRL, ROWS,
                                                  0xF, ROWS == 0xF);
  return (long long)(((uint64_t)hi << 32) | lo);
}
__device__ __forceinline__ long long wave_prefix(long long v) {
  v = v + dpp_i64<0x111>(v);
  v = v + dpp_i64<0x112>(v);
  v = v + dpp_i64<0x114>(v);
  v = v + dpp_i64<0x118>(v);
  v = v + dpp_i64<0x142, 0xA>(v);
  return v + dpp_i64<0x143, 0xC>(v);
}
__device__ __forceinline__ long long readlane_i64(long long v, int lane) {
  const uint32_t lo = __builtin_amdgcn_readlane((int)(uint32_t)v, lane);
  const uint32_t hi = __builtin_amdgcn_readlane((int)(uint32_t)((uint64_t)v >> 32), lane);
  return (long long)(((uint64_t)hi << 32) | lo);
}

// A thread's place in a sum over the block's W waves: what those in front of it have, and all.
struct Place {
  long long before, total;
};
template <int W>
__device__ __forceinline__ Place place_of(long long mine) {
  __shared__ long long wave_sum_[W];
  const int lane = threadIdx.x & 63, wave = same((int)threadIdx.x >> 6);
  const long long upto = wave_prefix(mine);
  if (lane == 63) wave_sum_[wave] = upto;
  __syncthreads();
  Place r = {upto - mine, 0};
  for (int w = 0; w < W; ++w) {
    if (w < wave) r.before += wave_sum_[w];
    r.total += wave_sum_[w];
  }
  r.total = same(r.total);
  return r;
}

// The tile of the share's sequence that holds a place in its ticks.
template <int HD, int C>
__device__ __forceinline__ void find_tile(const AttentionArgs& a, Share& r, long long at) {
  for (r.tile = 0;; ++r.tile) {
    const int ticks = kStart + same(tile_steps<HD, C>(a, r.rows, r.tile));
    if (at < ticks) break;
    at -= ticks;
  }
  r.at = (int)at;
}

// The beginnings of the shares of a block's WORKERS workers (4 waves, or the block): a thread sums
// the ticks of a run of tiles, and the one whose run holds the beginning finds its place. Sequences
// of few tiles are dealt out to the threads.
template <int HD, int C, int WORKERS>
__device__ __forceinline__ Share find_share_by_sequence(const AttentionArgs& a) {
  __shared__ int seq_[WORKERS];
  __shared__ long long at_[WORKERS];
  const int tid = threadIdx.x, n = a.batch.n_seqs, per = (n + 255) / 256;
  const int first = WORKERS * (int)blockIdx.x, own = WORKERS > 1 ? same(tid >> 6) : 0;
  const int s0 = tid * per, s1 = s0 + per < n ? s0 + per : n;
  auto ticks_of = [&](int s) {
    const Seq q = seq_of(a, s);
    long long n = 0;
    for (int t = 0; t * C < q.columns; ++t) n += kStart + tile_steps<HD, C>(a, q, t);
    return n;
  };
  long long mine = 0;
  for (int s = s0; s < s1; ++s) mine += ticks_of(s);
  const Place p = place_of<4>(mine);
  Share r = Share::of(a, p.total, first + own);
  for (int w = 0; w < WORKERS; ++w) {
    const int team = (first + w) / a.n_kv_heads;
    long long left = r.begin_of(team) - p.before;
    if (team < r.teams && left >= 0 && left < mine) {
      int s = s0;
      for (; s < s1 - 1; ++s) {
        const long long ticks = ticks_of(s);
        if (left < ticks) break;
        left -= ticks;
      }
      seq_[w] = s;
      at_[w] = left;
    }
  }
  __syncthreads();
  r.seq = same(seq_[own]);
  if (r.begin < r.end) {
    r.rows = same(seq_of(a, r.seq));
    find_tile<HD, C>(a, r, same(at_[own]));
  }
  return r;
}

// The same by each wave for itself, with up to 256 sequences in its lanes: no barrier, and the
// found one's rows come from its lane (one sequence 10.4 -> 9.4 us, 48 of up to 5 rows 35.3 ->
// 34.1).
template <int HD, int C>
__device__ __forceinline__ Share find_share_by_lane(const AttentionArgs& a, int worker) {
  constexpr int N = 4;
  const int lane = threadIdx.x & 63;
  Seq q[N];
  long long mine[N], upto[N], total = 0;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int s = 64 * i + lane;
    mine[i] = 0;
    q[i] = Seq{};
    if (64 * i >= a.batch.n_seqs) continue;
    if (s < a.batch.n_seqs) {
      q[i] = seq_of(a, s);
      for (int t = 0; t * C < q[i].columns; ++t) mine[i] += kStart + tile_steps<HD, C>(a, q[i], t);
    }
  }
#pragma unroll
  for (int i = 0; i < N; ++i) {
    upto[i] = 0;
    if (64 * i >= a.batch.n_seqs) continue;
    upto[i] = total + wave_prefix(mine[i]);
    total = readlane_i64(upto[i], 63);
  }
  Share r = Share::of(a, total, worker);
  if (r.begin >= r.end) return r;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const long long from = upto[i] - mine[i];
    const uint64_t at = __builtin_amdgcn_ballot_w64(r.begin >= from && r.begin < upto[i]);
    if (at) {
      const int l = __builtin_ctzll(at);
      r.seq = 64 * i + l;
      r.rows.row0 = __builtin_amdgcn_readlane(q[i].row0, l);
      r.rows.columns = __builtin_amdgcn_readlane(q[i].columns, l);
      r.rows.before = readlane_i64(q[i].before, l);
      r.rows.limit = readlane_i64(q[i].limit, l);
      find_tile<HD, C>(a, r, r.begin - readlane_i64(from, l));
    }
  }
  return r;
}

// One sequence of up to 256 tiles: a lane for each, 4 times (1507 rows 67.5 -> 65.7 us).
template <int HD, int C>
__device__ __forceinline__ Share find_share_of_one(const AttentionArgs& a, const Seq& q,
                                                   int worker) {
  constexpr int N = 4;
  const int lane = threadIdx.x & 63, tiles = (q.columns + C - 1) / C;
  long long mine[N], upto[N], total = 0;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int t = 64 * i + lane;
    mine[i] = upto[i] = 0;
    if (64 * i >= tiles) continue;
    if (t < tiles) mine[i] = kStart + tile_steps<HD, C>(a, q, t);
    upto[i] = total + wave_prefix(mine[i]);
    total = readlane_i64(upto[i], 63);
  }
  Share r = Share::of(a, total, worker);
  r.rows = q;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const long long from = upto[i] - mine[i];
    const uint64_t at =
        __builtin_amdgcn_ballot_w64(r.begin >= from && r.begin < upto[i] && r.begin < r.end);
    if (at) {
      const int l = __builtin_ctzll(at);
      r.tile = 64 * i + l;
      r.at = (int)(r.begin - readlane_i64(from, l));
    }
  }
  return r;
}

// Of those that have many each thread takes an equal part, whose beginning is looked up among the
// threads' sums of tiles (by sequence, where there is one of 1507 rows: 12.3 us, and 4.2 so).
template <int HD, int C, int W>
__device__ __forceinline__ Share find_share_by_tile(const AttentionArgs& a) {
  constexpr int T = 64 * W;
  __shared__ int upto_[T], found_[3];
  const int tid = threadIdx.x, n = a.batch.n_seqs, per = (n + T - 1) / T;
  int s0 = tid * per < n ? tid * per : n;
  int tiles_here = 0;
  for (int s = s0; s < s0 + per && s < n; ++s) tiles_here += (seq_of(a, s).columns + C - 1) / C;
  const Place q = place_of<W>(tiles_here);
  upto_[tid] = (int)q.before + tiles_here;
  __syncthreads();
  const int all = (int)q.total, each = all / T, more = all % T;
  const int tiles = each + (tid < more ? 1 : 0);
  int tile0 = each * tid + (tid < more ? tid : more);
  int lo = 0;  // the thread whose sequences have tile0
  for (int d = T / 2; d > 0; d /= 2)
    if (upto_[lo + d - 1] <= tile0) lo += d;
  if (lo > 0) tile0 -= upto_[lo - 1];
  s0 = lo * per;
  // each tile of the run in turn, until `what` says that it is enough
  auto run = [&](auto what) {
    int left = tiles, t = tile0;
    for (int s = s0; s < n && left > 0; ++s) {
      const Seq q = seq_of(a, s);
      for (; t * C < q.columns && left > 0; ++t, --left)
        if (what(s, t, kStart + tile_steps<HD, C>(a, q, t))) return;
      t -= (q.columns + C - 1) / C;
    }
  };
  long long mine = 0;
  run([&](int, int, int ticks) {
    mine += ticks;
    return false;
  });
  const Place p = place_of<W>(mine);
  Share r = Share::of(a, p.total, blockIdx.x);
  long long left = r.begin - p.before;
  if (r.begin < r.end && left >= 0 && left < mine)
    run([&](int s, int t, int ticks) {
      if (left >= ticks) {
        left -= ticks;
        return false;
      }
      found_[0] = s;
      found_[1] = t;
      found_[2] = (int)left;
      return true;
    });
  __syncthreads();
  r.seq = same(found_[0]);
  r.tile = same(found_[1]);
  r.at = same(found_[2]);
  if (r.begin < r.end) r.rows = same(seq_of(a, r.seq));
  return r;
}

// x, or -inf where bit i is set: without a comparison's scalar registers, which a step has none to
// spare of.
__device__ __forceinline__ float hide(float x, uint32_t bits, int i) {
  const uint32_t m = (uint32_t)__builtin_amdgcn_sbfe((int)bits, i, 1);
  return __builtin_bit_cast(float, (m & 0xFF800000u) | (~m & __builtin_bit_cast(uint32_t, x)));
}

// The larger of x and what the lane 16 (32) away has.
__device__ __forceinline__ float max_across(float x, bool halves) {
  const uint32_t b = __builtin_bit_cast(uint32_t, x);
  const auto r = halves ? __builtin_amdgcn_permlane32_swap(b, b, false, false)
                        : __builtin_amdgcn_permlane16_swap(b, b, false, false);
  const uint32_t r0 = r[0], r1 = r[1];
  return __builtin_fmaxf(__builtin_bit_cast(float, r0), __builtin_bit_cast(float, r1));
}
__device__ __forceinline__ float max_of_quarters(float x) {
  return max_across(max_across(x, false), true);
}

// Units of few columns, a wave each. With C = 16 QT columns (rows x heads of the group) a step is
//   S^T = K Q^T   (v_mfma_f32_16x16x32_f16; A: 16 positions of K, B: 16 columns of q)
//   O^T += V^T P^T (.._bf16; A: 16 dims of V, B: the lane's own weights)
// and no operand changes lanes: lane (n = l % 16, qd = l / 16) gets of S^T column n, positions 4 qd
// .. 4 qd + 3 of each page, and those positions, of two pages, are its places in the second
// product's contraction. K is loaded 16 bytes a lane (position n, dims 16 qd ..): the order of dims
// in the contraction is free, and q is loaded in it too. V is loaded 4 (8) bytes for each of 4
// positions; dims 4 n .. become the rows n of 4 (8) products, so that a lane ends with 16 (32) dims
// in a row. Nothing goes through LDS and no wave waits for another. A step's K is loaded when the
// last one's is used up and its V likewise, 8 KiB on the way for each SIMD; steps of twice the size
// 59.8 -> 65.1 us (256 sequences), 50.5 -> 53.1 (3 long ones). Bound by HBM: 55 us of 256
// sequences' 59 for 283 MB, the rest is the joining launch; of a single short sequence's 9.4 us 6.7
// are the way from the lengths over the table and the scales to K and V, one load behind the other.
template <int HD, int QT>
__global__ void __launch_bounds__(256, 2) k_kv8_attention_few(const AttentionArgs a) {
  constexpr int C = 16 * QT, KU = HD / 64, VW = HD / 64, PG = kPages<HD, C>, STEP = kStep<HD, C>;
  const int lane = threadIdx.x & 63, n = lane & 15, qd = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int worker = 4 * (int)blockIdx.x + wave;
  const bool shared_units = a.parts != nullptr;
  const Share sh = a.batch.n_seqs <= 256 ? find_share_by_lane<HD, C>(a, worker)
                                         : find_share_by_sequence<HD, C, 4>(a);
  const int h = sh.head;
  auto note = [&](int side, int first, int last, int column, int columns, const Seq& q) {
    Shared o = {};
    o.first = first;
    o.last = last;
    o.column = column;
    o.columns = columns;
    o.row0 = q.row0;
    o.blind = blind_of(a, q);
    if (lane == 0) a.shared[2 * worker + side] = o;
  };
  if (shared_units) {
    note(0, 0, -1, 0, 0, Seq{});
    note(1, 0, -1, 0, 0, Seq{});
  }

  long long pos = sh.begin;
  if (pos < sh.end) {
    int s = sh.seq, tile = sh.tile, tick = sh.at;
    Seq q = sh.rows;
    int steps = same(tile_steps<HD, C>(a, q, tile));
    const float to_log2 = kLog2e / __builtin_sqrtf((float)HD);
    int ids = 0, ids_of = -1, window = -1;  // 64 entries of a sequence's table, one to a lane

    while (pos < sh.end) {
      const int ticks = kStart + steps;
      int upto = ticks;  // this worker's end of the unit
      if (shared_units && sh.end - pos < ticks - tick) upto = tick + (int)(sh.end - pos);
      const int step = tick > kStart ? tick - kStart : 0;
      int stop = upto > kStart ? upto - kStart : 0;
      pos += upto - tick;
      // without a workspace, a unit that began in the share before is done there
      if (stop > step && (shared_units || tick == 0)) {
        stop = same(stop);
        const int c0 = tile * C;
        const int columns = q.columns - c0 < C ? q.columns - c0 : C;
        const int see_max = same(seen(a, q, c0 + columns - 1)), see_min = same(seen(a, q, c0));

        int see[QT];
        f16x8 qf[QT][2 * KU];
#pragma unroll
        for (int t = 0; t < QT; ++t) {
          const int c = 16 * t + n;
          const bool own = c < columns;
          const int col = c0 + (own ? c : 0);
          see[t] = own ? seen(a, q, col) : 0;
          const size_t row = q.row0 + col / a.group;
          const f16* src = a.q + (row * a.n_heads + h * a.group + col % a.group) * HD + 16 * qd;
#pragma unroll
          for (int u = 0; u < 2 * KU; ++u)
            qf[t][u] = own ? as_h8(ld16(src + 64 * (u / 2) + 8 * (u % 2))) : (f16x8)(f16)0;
        }
        f32x4 acc[QT][4 * VW];
        float m[QT];
        Sum l[QT];
#pragma unroll
        for (int t = 0; t < QT; ++t) {
          m[t] = -INFINITY;
          l[t] = Sum{0.0f, 0.0f};
#pragma unroll
          for (int c = 0; c < 4 * VW; ++c) acc[t][c] = f32x4{0, 0, 0, 0};
        }

        const int* pages = a.batch.tables + (size_t)s * a.batch.max_pages;
        if (see_max > 0) {
          // their scales for this head
          float ksc, vsc;
          const int last_page = (int)((q.limit + kPage - 1) / kPage) - 1;
          auto load_ids = [&] {
            const int p = 64 * window + lane;
            ids = pages[p < last_page ? p : last_page];
          };
          u32x4 kr[PG][KU];
          uint32_t vr[PG][4][VW];
          float ks[PG], vs[PG], vs_next[PG];
          const uint8_t* v_next[PG];
          auto load_scales = [&] {
            const size_t b = (size_t)ids * a.n_kv_heads + h;
            ksc = a.k_scale[b];
            vsc = a.v_scale[b];
          };
          // the pages of a step: loads of K, and where V is
          auto load_k = [&](int st) {
#pragma unroll
            for (int p = 0; p < PG; ++p) {
              const int i = (PG * st + p) & 63;
              const size_t at = ((size_t)__builtin_amdgcn_readlane(ids, i) * a.n_kv_heads + h) *
                                (size_t)(kPage * HD);
              const uint8_t* src = a.k_pool + at;
#pragma unroll
              for (int u = 0; u < KU; ++u)
                kr[p][u] = ld16_stream(src + (uint32_t)(n * HD + 16 * qd + 64 * u));
              v_next[p] = a.v_pool + at;
            }
          };
          auto take_scales = [&](int st) {
#pragma unroll
            for (int p = 0; p < PG; ++p) {
              const int i = (PG * st + p) & 63;
              ks[p] = readlane_f32(ksc, i);
              vs_next[p] = readlane_f32(vsc, i);
            }
          };
          auto load_v = [&] {
#pragma unroll
            for (int p = 0; p < PG; ++p) {
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                const uint8_t* src = v_next[p] + (uint32_t)((4 * qd + i) * HD + 4 * VW * n);
                if constexpr (VW == 1) {
                  vr[p][i][0] = __builtin_nontemporal_load(reinterpret_cast<const uint32_t*>(src));
                } else {
                  const u32x2 x = __builtin_nontemporal_load(reinterpret_cast<const u32x2*>(src));
                  vr[p][i][0] = x[0];
                  vr[p][i][VW - 1] = x[1];
                }
              }
            }
          };
          // MORE: another step of the unit follows, whose K is loaded when this one's is used up,
          // and its V likewise. (A load that may or may not happen would make the waits for those
          // in front of it as strict as if it did not.)
          auto one_step = [&](int st, auto more) {
            constexpr bool MORE = decltype(more)::value;
            const bool edge = (st + 1) * STEP > see_min;  // some row does not see all of it
            f32x4 sc[QT][PG];
#pragma unroll
            for (int t = 0; t < QT; ++t)
#pragma unroll
              for (int p = 0; p < PG; ++p) sc[t][p] = f32x4{0, 0, 0, 0};
#pragma unroll
            for (int p = 0; p < PG; ++p)
#pragma unroll
              for (int u = 0; u < 2 * KU; ++u) {
                const uint32_t lo = elem(kr[p][u / 2], 2 * (u % 2));
                const uint32_t hi = elem(kr[p][u / 2], 2 * (u % 2) + 1);
                u32x4 w;
                w[0] = __builtin_bit_cast(uint32_t, from_e4m3<false>(lo, ks[p]));
                w[1] = __builtin_bit_cast(uint32_t, from_e4m3<true>(lo, ks[p]));
                w[2] = __builtin_bit_cast(uint32_t, from_e4m3<false>(hi, ks[p]));
                w[3] = __builtin_bit_cast(uint32_t, from_e4m3<true>(hi, ks[p]));
#pragma unroll
                for (int t = 0; t < QT; ++t)
                  sc[t][p] = __builtin_amdgcn_mfma_f32_16x16x32_f16(as_h8(w), qf[t][u], sc[t][p],
                                                                    0, 0, 0);
              }
            if constexpr (MORE) {
              if ((st + 1) * PG / 64 != window) {
                window = (st + 1) * PG / 64;
                load_ids();
                load_scales();
                // waited for here: later, the loads of K and V behind them would be, too
                asm volatile("" : "+v"(ids), "+v"(ksc), "+v"(vsc));
              }
              load_k(st + 1);
              take_scales(st + 1);
            }
            const int key0 = st * STEP + 4 * qd;
            uint32_t ph[QT][PG][2], pl[QT][PG][2];
#pragma unroll
            for (int t = 0; t < QT; ++t) {
              if (edge) {
                const int left = see[t] - key0;
#pragma unroll
                for (int p = 0; p < PG; ++p) {
#pragma unroll
                  for (int i = 0; i < 4; ++i)
                    if (16 * p + i >= left) sc[t][p][i] = -INFINITY;
                  asm volatile("" : "+v"(sc[t][p]));  // here: a branch, not selects in every step
                }
              }
              float top = -INFINITY;
#pragma unroll
              for (int p = 0; p < PG; ++p)
#pragma unroll
                for (int i = 0; i < 4; ++i) top = __builtin_fmaxf(top, sc[t][p][i]);
              top = max_of_quarters(top) * to_log2;
              const float next = top > m[t] + kSlack ? top : m[t];
              const float ref = next == -INFINITY ? 0.0f : next;
              if (__builtin_amdgcn_ballot_w64(next != m[t])) {
                const float corr = __builtin_amdgcn_exp2f(m[t] - ref);
                l[t].scale(corr);
#pragma unroll
                for (int c = 0; c < 4 * VW; ++c) acc[t][c] = acc[t][c] * corr;
                m[t] = next;
              }
              float scale = to_log2;
              if (__builtin_amdgcn_ballot_w64(__builtin_fabsf(ref) >= kLargeScore)) {
                scale = 1.0f;
#pragma unroll
                for (int p = 0; p < PG; ++p) {
                  sc[t][p] = sc[t][p] * to_log2;
                  asm volatile("" : "+v"(sc[t][p]));
                }
              }
              float sum = 0.0f;
#pragma unroll
              for (int p = 0; p < PG; ++p)
#pragma unroll
                for (int i = 0; i < 4; i += 2) {
                  const float w0 =
                      __builtin_amdgcn_exp2f(__builtin_fmaf(sc[t][p][i], scale, -ref));
                  const float w1 =
                      __builtin_amdgcn_exp2f(__builtin_fmaf(sc[t][p][i + 1], scale, -ref));
                  sum = sum + (w0 + w1);
                  split_rounded(w0, w1, ph[t][p][i / 2], pl[t][p][i / 2]);
                }
              l[t].add(sum);
            }
            if (edge) {
              // What no row sees is stale: zero. A NaN of a position that only some rows see would
              // reach the others through their zero weights: it is taken out and handed to its
              // rows.
              uint32_t odd = 0;
#pragma unroll
              for (int p = 0; p < PG; ++p)
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                  for (int w = 0; w < VW; ++w) {
                    const uint32_t b = key0 + 16 * p + i < see_max ? vr[p][i][w] : 0u;
                    const uint32_t bad = ((b & 0x7F7F7F7Fu) + 0x01010101u) & 0x80808080u;
                    odd |= bad;
                    vr[p][i][w] = b & ~((bad >> 7) * 0xFFu);
                  }
              if (__builtin_amdgcn_ballot_w64(odd != 0)) {
                for (int key = st * STEP; key < (st + 1) * STEP && key < see_max; ++key) {
                  const size_t b = (size_t)pages[key / kPage] * a.n_kv_heads + h;
                  const uint8_t* src =
                      a.v_pool + (b * kPage + key % kPage) * HD + 16 * VW * qd;
#pragma unroll
                  for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int w = 0; w < VW; ++w) {
                      const uint32_t x = reinterpret_cast<const uint32_t*>(src)[VW * i + w];
#pragma unroll
                      for (int c = 0; c < 4; ++c)
#pragma unroll
                        for (int t = 0; t < QT; ++t) {
                          const bool bad = key < see[t] && ((x >> (8 * c)) & 0x7Fu) == 0x7Fu;
                          f32x4& o = acc[t][4 * w + c];
                          o[i] = bad ? __builtin_nanf("") : o[i];
                        }
                    }
                }
              }
            }
#pragma unroll
            for (int pp = 0; pp < PG; pp += 2)
#pragma unroll
              for (int w = 0; w < VW; ++w)
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                  constexpr uint32_t sel[2] = {0x05010400u, 0x07030602u};
                  const uint32_t a01 =
                      __builtin_amdgcn_perm(vr[pp][1][w], vr[pp][0][w], sel[half]);
                  const uint32_t a23 =
                      __builtin_amdgcn_perm(vr[pp][3][w], vr[pp][2][w], sel[half]);
                  const uint32_t b01 =
                      __builtin_amdgcn_perm(vr[pp + 1][1][w], vr[pp + 1][0][w], sel[half]);
                  const uint32_t b23 =
                      __builtin_amdgcn_perm(vr[pp + 1][3][w], vr[pp + 1][2][w], sel[half]);
#pragma unroll
                  for (int c = 0; c < 2; ++c) {
                    auto two = [&](uint32_t b, float scale) {
                      return c ? bf16_from_e4m3<true>(b, scale) : bf16_from_e4m3<false>(b, scale);
                    };
                    const u32x4 v4 = {two(a01, vs[pp]), two(a23, vs[pp]), two(b01, vs[pp + 1]),
                                      two(b23, vs[pp + 1])};
                    const bf16x8 vf = __builtin_bit_cast(bf16x8, v4);
#pragma unroll
                    for (int t = 0; t < QT; ++t) {
                      const u32x4 h4 = {ph[t][pp][0], ph[t][pp][1], ph[t][pp + 1][0],
                                        ph[t][pp + 1][1]};
                      const u32x4 l4 = {pl[t][pp][0], pl[t][pp][1], pl[t][pp + 1][0],
                                        pl[t][pp + 1][1]};
                      f32x4& o = acc[t][4 * w + 2 * half + c];
                      o = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
                          vf, __builtin_bit_cast(bf16x8, h4), o, 0, 0, 0);
                      o = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
                          vf, __builtin_bit_cast(bf16x8, l4), o, 0, 0, 0);
                    }
                  }
                }
            if constexpr (MORE) {
              load_v();
#pragma unroll
              for (int p = 0; p < PG; ++p) vs[p] = vs_next[p];
            }
          };
          if (s != ids_of || step * PG / 64 != window) {
            window = step * PG / 64;
            ids_of = s;
            load_ids();
          }
          load_scales();
          load_k(step);
          load_v();
          take_scales(step);
#pragma unroll
          for (int p = 0; p < PG; ++p) vs[p] = vs_next[p];
          int st = step;
          for (; st < stop - 1; ++st) one_step(st, std::true_type{});
          one_step(st, std::false_type{});
        }

        const bool whole = step == 0 && stop == steps;
        const int side = step == 0 ? 1 : 0;
        if (!whole) {  // the workers of its first and last steps
          const long long end = pos + ticks - upto, begin = end - steps;
          note(side, sh.team_at(begin), sh.team_at(end - 1), c0, columns, q);
        }
        const size_t slot = 2 * (size_t)worker + side;
#pragma unroll
        for (int t = 0; t < QT; ++t) {
          float sum = l[t].of + __shfl_xor(l[t].of, 16);
          sum = sum + __shfl_xor(sum, 32);
          const int c = 16 * t + n;
          if (c >= columns) continue;
          if (whole) {
            const int col = c0 + c;
            f16* dst = a.out + ((size_t)(q.row0 + col / a.group) * a.n_heads + h * a.group +
                                col % a.group) * HD + 16 * VW * qd;
#pragma unroll
            for (int g = 0; g < 2 * VW; ++g) {
              f16x8 o;
#pragma unroll
              for (int e = 0; e < 8; ++e) {
                const int d = 8 * g + e;  // of this lane's dims: (i, chunk)
                const float y = acc[t][d % (4 * VW)][d / (4 * VW)];
                o[e] = see[t] > 0 ? (f16)(y / sum) : (f16)0;
              }
              st16(dst + 8 * g, as_u4(o));
            }
          } else {
            float* dst = a.parts + (slot * C + c) * HD + 16 * VW * qd;
#pragma unroll
            for (int g = 0; g < 4 * VW; ++g) {
              f32x4 o;
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                const int d = 4 * g + e;
                o[e] = acc[t][d % (4 * VW)][d / (4 * VW)];
              }
              *reinterpret_cast<f32x4*>(dst + 4 * g) = o;
            }
            if (qd == 0) a.parts_ml[slot * C + c] = make_float2(m[t], sum);
          }
        }
      }
      tick = 0;
      ++tile;
      while (tile * C >= q.columns && s < a.batch.n_seqs - 1) {
        tile = 0;
        q = same(seq_of(a, ++s));
      }
      if (tile * C >= q.columns) break;
      steps = same(tile_steps<HD, C>(a, q, tile));
    }
  }
}

// Joins the parts of units: the one that a unit's first worker left (an odd slot) and those of the
// workers behind it (even slots). Block (b, y) looks at the units that worker b has a part in, at
// the y-th 256 of their tasks (a column's 4 dims). The n workers of a unit share them among their
// blocks, in up to n / 4 slices, and a block deals the parts out over the threads that a slice
// leaves, which meet in LDS. Bound by latency where rows are few, 3.7 us of a trace for one
// sequence and 4.7 for 256, and by the parts' bytes for prompts: 8.6 us for the 20 MB, written and
// read, of 1507 rows.
template <int HD>
__global__ void __launch_bounds__(256) k_kv8_attention_join(const AttentionArgs a, int C) {
  constexpr int V = HD / 4;
  __shared__ f32x4 others[256];
  __shared__ float2 others_ml[256];
  const int tid = threadIdx.x, worker = blockIdx.x;
  struct Joint {
    f32x4 acc;
    float m, l;
    __device__ __forceinline__ void add(f32x4 x, float2 ml) {
      const float next = __builtin_fmaxf(m, ml.x), ref = next == -INFINITY ? 0.0f : next;
      const float wa = __builtin_amdgcn_exp2f(m - ref), wb = __builtin_amdgcn_exp2f(ml.x - ref);
      acc = acc * wa + x * wb;
      l = l * wa + ml.y * wb;
      m = next;
    }
  };
  const int team = worker / a.n_kv_heads, head = worker % a.n_kv_heads;
  const Shared both[2] = {a.shared[2 * worker], a.shared[2 * worker + 1]};
#pragma unroll
  for (int side = 0; side < 2; ++side) {
    const Shared o = both[side];
    if (!is_unit(o, team, a.teams, C)) continue;
    const int n = o.last - o.first + 1, base = 256 * blockIdx.y;
    const int tasks = V * o.columns - base < 256 ? V * o.columns - base : 256;
    if (tasks <= 0) continue;
    int lanes = 16, slices = 1;  // tasks of a slice
    while (lanes < tasks) lanes *= 2;
    while (8 * slices <= n && lanes > 16) {
      slices *= 2;
      lanes /= 2;
    }
    const int slice = team - o.first;
    if (slice >= slices) continue;
    const int deal = 256 / lanes, turn = tid / lanes;
    const int task = base + slice * lanes + tid % lanes, c = task / V, d = 4 * (task % V);
    Joint r = {f32x4{0, 0, 0, 0}, -INFINITY, 0.0f};
    if (c < o.columns) {
#pragma unroll 4
      for (int j = turn; j < n; j += deal) {
        const size_t w = (size_t)(o.first + j) * a.n_kv_heads + head;
        const size_t at = (2 * w + (j == 0 ? 1 : 0)) * C + c;
        r.add(*reinterpret_cast<const f32x4*>(a.parts + at * HD + d), a.parts_ml[at]);
      }
    }
    __syncthreads();
    others[tid] = r.acc;
    others_ml[tid] = make_float2(r.m, r.l);
    __syncthreads();
    if (turn == 0 && c < o.columns) {
      for (int k = 1; k < deal && k < n; ++k)
        r.add(others[tid + k * lanes], others_ml[tid + k * lanes]);
      const int col = o.column + c, row = row_of(o, c, a.batch.n_rows, a.group);
      const bool any = col >= o.blind;
      f16x2 y[2];
#pragma unroll
      for (int e = 0; e < 4; ++e) y[e / 2][e % 2] = any ? (f16)(r.acc[e] / r.l) : (f16)0;
      uint2 v;
      v.x = __builtin_bit_cast(uint32_t, y[0]);
      v.y = __builtin_bit_cast(uint32_t, y[1]);
      if (row >= 0)
        *reinterpret_cast<uint2*>(
            a.out + ((size_t)row * a.n_heads + head * a.group + col % a.group) * HD + d) = v;
    }
  }
}

// Units of many columns, a block each: W = 4 or 8 waves of 32 columns share the K and V of a step
// through LDS, where they arrive as fp16 and bf16 (each wave converts its part). Per wave
//   S^T = K Q^T    (v_mfma_f32_32x32x16_f16; A: 32 positions of K, B: 32 columns of q)
//   O^T += V^T P^T (.._bf16; A: 32 dims of V, B: the lane's own weights)
// Lane l gets of S^T column l % 32, positions 8 (i / 4) + 4 (l / 32) + i % 4; V's positions lie in
// LDS in the order in which that makes 8 of them a lane's share of a contraction. Two buffers and a
// barrier a step; the next but one's loads are on their way meanwhile. 1507 rows: 65 us, of which
// a block is 2 on the way to its share, 3 on that to its first step's data, 47 in its 14 steps and
// 2 writing parts; the joining launch and the gap in front of it take the rest.
template <int HD, int W>
__global__ void __launch_bounds__(64 * W, 2) k_kv8_attention_many(const AttentionArgs a) {
  constexpr int C = 32 * W, PG = kPages<HD, C>, STEP = kStep<HD, C>, KT = STEP / 32, DT = HD / 32;
  constexpr int KP = HD / 16, VP = HD / 4;  // threads to a position of K, to 4 positions of V
  // One piece of 16 bytes behind each row: 16 lanes that read a piece of as many rows meet no bank
  // twice, and every address is a lane's base and a constant. Rows change places within 16 so that
  // neither do lanes that write: K's come 4 (2) at a time, and V's are 4 apart.
  __shared__ u32x4 k_lds[2][STEP][HD / 8 + 1];  // [position][8 dims]
  __shared__ u32x4 v_lds[2][HD][STEP / 8 + 1];  // [dim][8 positions]
  __shared__ int odd[2];  // a NaN was taken out of V: of a unit, and of the next
  const int tid = threadIdx.x, lane = tid & 63, n = lane & 31, half = lane >> 5;
  const int wave = same(tid >> 6), worker = blockIdx.x;
  auto k_row = [](int key) {
    return (key & ~15) | ((key & 2) << 2) | ((key & 12) >> 1) | (key & 1);
  };
  auto v_row = [](int d) { return (d & ~15) | ((d + (d >> 4)) & 15); };
  const bool shared_units = a.parts != nullptr;
  int turn = 0;
  if (tid < 2) odd[tid] = 0;
  Share sh;
  const Seq one = same(seq_of(a, 0));
  if (a.batch.n_seqs == 1 && one.columns <= 256 * C)
    sh = find_share_of_one<HD, C>(a, one, worker);
  else if constexpr (W == 8)
    sh = find_share_by_tile<HD, C, W>(a);
  else
    sh = a.batch.n_seqs <= 256 ? find_share_by_lane<HD, C>(a, worker)
                               : find_share_by_sequence<HD, C, 1>(a);
  const int h = sh.head;
  auto note = [&](int side, int first, int last, int column, int columns, const Seq& q) {
    Shared o = {};
    o.first = first;
    o.last = last;
    o.column = column;
    o.columns = columns;
    o.row0 = q.row0;
    o.blind = blind_of(a, q);
    if (tid == 0) a.shared[2 * worker + side] = o;
  };
  if (shared_units) {
    note(0, 0, -1, 0, 0, Seq{});
    note(1, 0, -1, 0, 0, Seq{});
  }
  long long pos = sh.begin;
  if (pos >= sh.end) return;
  int s = sh.seq, tile = sh.tile, tick = sh.at;
  Seq q = sh.rows;
  int steps = same(tile_steps<HD, C>(a, q, tile));
  const float to_log2 = kLog2e / __builtin_sqrtf((float)HD);

  while (pos < sh.end) {
    const int ticks = kStart + steps;
    int upto = ticks;  // this worker's end of the unit
    if (shared_units && sh.end - pos < ticks - tick) upto = tick + (int)(sh.end - pos);
    const int step = tick > kStart ? tick - kStart : 0;
    const int stop = same(upto > kStart ? upto - kStart : 0);
    pos += upto - tick;
    if (stop > step && (shared_units || tick == 0)) {
      const int c0 = tile * C;
      const int columns = q.columns - c0 < C ? q.columns - c0 : C;
      const int see_max = same(seen(a, q, c0 + columns - 1)), see_min = same(seen(a, q, c0));
      const int* pages = a.batch.tables + (size_t)s * a.batch.max_pages;
      const int last_page = (int)((q.limit + kPage - 1) / kPage) - 1;

      // this wave's columns
      const int first_own = 32 * wave, c = first_own + n;
      const bool own = c < columns;
      const int col = c0 + (own ? c : 0);
      const int see = own ? seen(a, q, col) : 0;
      const int last_own = first_own + 31 < columns ? first_own + 31 : columns - 1;
      const int wave_max = first_own < columns ? same(seen(a, q, c0 + last_own)) : 0;
      const int wave_min = first_own + 31 < columns ? same(seen(a, q, c0 + first_own)) : 0;
      const f16* src = a.q + ((size_t)(q.row0 + col / a.group) * a.n_heads + h * a.group +
                              col % a.group) * HD + 8 * half;
      f16x8 qf[HD / 16];
#pragma unroll
      for (int u = 0; u < HD / 16; ++u) qf[u] = own ? as_h8(ld16(src + 16 * u)) : (f16x8)(f16)0;
      float m = -INFINITY;
      Sum sum = {0.0f, 0.0f};
      f32x16 acc[DT];
#pragma unroll
      for (int d = 0; d < DT; ++d)
#pragma unroll
        for (int i = 0; i < 16; ++i) acc[d][i] = 0.0f;

      if (see_max > 0) {
        // 64 table entries, one to a lane, and their scales; the wave's page of a step on its way
        int window = -1, ids = 0;
        float ksc = 0, vsc = 0, ks = 0, vs = 0;
        u32x4 kr;
        uint32_t vr[4];
        const int k_key = tid / KP, k_part = tid % KP, v_part = tid % VP;
        // 4 positions of V; those of a wave fill both halves of a piece
        const int vt = VP == 16 ? tid / VP : 4 * (wave / 2) + (wave & 1) + 2 * (lane / VP);
        const int v_key = 4 * vt;
        auto load = [&](int st) {
          const int w = st * PG / 64;
          if (w != window) {
            window = w;
            const int p = 64 * w + lane;
            ids = pages[p < last_page ? p : last_page];
            const size_t b = (size_t)ids * a.n_kv_heads + h;
            ksc = a.k_scale[b];
            vsc = a.v_scale[b];
          }
          const int i = (PG * st + wave * PG / W) & 63;  // the page of this wave's part
          const size_t block = ((size_t)__builtin_amdgcn_readlane(ids, i) * a.n_kv_heads + h) *
                               (size_t)(kPage * HD);
          kr = ld16(a.k_pool + block + (uint32_t)(k_key % kPage * HD + 16 * k_part));
#pragma unroll
          for (int i4 = 0; i4 < 4; ++i4)
            vr[i4] = *reinterpret_cast<const uint32_t*>(
                a.v_pool + block + (uint32_t)((v_key % kPage + i4) * HD + 4 * v_part));
          ks = readlane_f32(ksc, i);
          vs = readlane_f32(vsc, i);
        };
        auto store = [&](int st, int buf) {
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const uint32_t x = elem(kr, 2 * j), y = elem(kr, 2 * j + 1);
            u32x4 w;
            w[0] = __builtin_bit_cast(uint32_t, from_e4m3<false>(x, ks));
            w[1] = __builtin_bit_cast(uint32_t, from_e4m3<true>(x, ks));
            w[2] = __builtin_bit_cast(uint32_t, from_e4m3<false>(y, ks));
            w[3] = __builtin_bit_cast(uint32_t, from_e4m3<true>(y, ks));
            k_lds[buf][k_row(k_key)][2 * k_part + j] = w;
          }
          if ((st + 1) * STEP > see_min) {
            // What no row sees is stale: zero. A NaN of a position that only some rows see would
            // reach the others through their zero weights: it is handed to its rows at the end.
            uint32_t bad = 0;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const uint32_t b = st * STEP + v_key + i < see_max ? vr[i] : 0u;
              const uint32_t x = ((b & 0x7F7F7F7Fu) + 0x01010101u) & 0x80808080u;
              bad |= x;
              vr[i] = b & ~((x >> 7) * 0xFFu);
            }
            if (bad) odd[turn] = 1;
          }
          const int piece = 2 * (vt / 4) + (vt & 1);
#pragma unroll
          for (int g = 0; g < 2; ++g) {
            constexpr uint32_t sel[2] = {0x05010400u, 0x07030602u};
            const uint32_t x01 = __builtin_amdgcn_perm(vr[1], vr[0], sel[g]);
            const uint32_t x23 = __builtin_amdgcn_perm(vr[3], vr[2], sel[g]);
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const int d = 4 * v_part + 2 * g + e;
              u32x2 y;
              y[0] = e ? bf16_from_e4m3<true>(x01, vs) : bf16_from_e4m3<false>(x01, vs);
              y[1] = e ? bf16_from_e4m3<true>(x23, vs) : bf16_from_e4m3<false>(x23, vs);
              reinterpret_cast<u32x2*>(&v_lds[buf][v_row(d)][piece])[(vt >> 1) & 1] = y;
            }
          }
        };
        auto compute = [&](int st, int buf) {
          // 4 pieces of K are on their way while 4 are multiplied: the compiler, left to itself,
          // waits for each (1507 rows: 69.6 us, and 67.0 so)
          constexpr int G = 4, GROUPS = KT * (HD / 16) / G;
          f32x16 sc[KT];
          u32x4 kf[2][G];
          auto fetch = [&](int g) {
#pragma unroll
            for (int j = 0; j < G; ++j) {
              const int u = (G * g + j) / KT, t = (G * g + j) % KT;
              kf[g & 1][j] = k_lds[buf][32 * t + k_row(n)][2 * u + half];
            }
          };
#pragma unroll
          for (int t = 0; t < KT; ++t)
#pragma unroll
            for (int i = 0; i < 16; ++i) sc[t][i] = 0.0f;
          fetch(0);
#pragma unroll
          for (int g = 0; g < GROUPS; ++g) {
            if (g + 1 < GROUPS) fetch(g + 1);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int j = 0; j < G; ++j) {
              const int u = (G * g + j) / KT, t = (G * g + j) % KT;
              sc[t] = __builtin_amdgcn_mfma_f32_32x32x16_f16(as_h8(kf[g & 1][j]), qf[u], sc[t], 0,
                                                             0, 0);
            }
          }
          if ((st + 1) * STEP > wave_min) {  // some row does not see all of it
#pragma unroll
            for (int t = 0; t < KT; ++t) {
              // of 8 positions in a row a lane has 4: the number of those that its row sees
              int left = see - (st * STEP + 32 * t + 4 * half);
              left = left < 0 ? 0 : left > 32 ? 32 : left;
              const uint32_t beyond = 0xFFFFu << (4 * (left / 8) + (left % 8 < 4 ? left % 8 : 4));
#pragma unroll
              for (int i = 0; i < 16; ++i) sc[t][i] = hide(sc[t][i], beyond, i);
              asm volatile("" : "+v"(sc[t]));  // here: a branch, not selects in every step
            }
          }
          float top = sc[0][0];
#pragma unroll
          for (int t = 0; t < KT; ++t)
#pragma unroll
            for (int i = 0; i < 16; ++i) top = __builtin_fmaxf(top, sc[t][i]);
          top = max_across(top, true) * to_log2;
          const float next = top > m + kSlack ? top : m;
          const float ref = next == -INFINITY ? 0.0f : next;
          if (__builtin_amdgcn_ballot_w64(next != m)) {
            const float corr = __builtin_amdgcn_exp2f(m - ref);
            sum.scale(corr);
#pragma unroll
            for (int d = 0; d < DT; ++d)
#pragma unroll
              for (int i = 0; i < 16; ++i) acc[d][i] = acc[d][i] * corr;
            m = next;
          }
          float scale = to_log2;
          if (__builtin_amdgcn_ballot_w64(__builtin_fabsf(ref) >= kLargeScore)) {
            scale = 1.0f;
#pragma unroll
            for (int t = 0; t < KT; ++t) {
#pragma unroll
              for (int i = 0; i < 16; ++i) sc[t][i] = sc[t][i] * to_log2;
              asm volatile("" : "+v"(sc[t]));
            }
          }
          float of_step = 0.0f;
#pragma unroll
          for (int cc = 0; cc < 2 * KT; ++cc) {  // 16 positions
            uint32_t ph[4], pl[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const int i = 8 * (cc % 2) + 2 * e;
              const float w0 =
                  __builtin_amdgcn_exp2f(__builtin_fmaf(sc[cc / 2][i], scale, -ref));
              const float w1 =
                  __builtin_amdgcn_exp2f(__builtin_fmaf(sc[cc / 2][i + 1], scale, -ref));
              of_step = of_step + (w0 + w1);
              split_cut(w0, w1, ph[e], pl[e]);
            }
            const bf16x8 hi = __builtin_bit_cast(bf16x8, (u32x4{ph[0], ph[1], ph[2], ph[3]}));
            const bf16x8 lo = __builtin_bit_cast(bf16x8, (u32x4{pl[0], pl[1], pl[2], pl[3]}));
#pragma unroll
            for (int d = 0; d < DT; ++d) {
              const bf16x8 vf = __builtin_bit_cast(bf16x8, v_lds[buf][v_row(32 * d + n)][2 * cc + half]);
              acc[d] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(vf, hi, acc[d], 0, 0, 0);
              acc[d] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(vf, lo, acc[d], 0, 0, 0);
            }
          }
          sum.add(of_step);
        };
        load(step);
        lds_barrier();  // the unit before is done with
        if (tid == 0) odd[turn ^ 1] = 0;
        store(step, 0);
        if (step + 1 < stop) load(step + 1);
        lds_barrier();
        for (int st = step; st < stop; ++st) {
          const int buf = (st - step) & 1;
          if (st * STEP < wave_max) compute(st, buf);
          if (st + 1 < stop) {
            store(st + 1, buf ^ 1);
            if (st + 2 < stop) load(st + 2);
          }
          lds_barrier();
        }
        if (odd[turn]) {
          int key = see_min / STEP * STEP;
          key = key > step * STEP ? key : step * STEP;
          for (; key < stop * STEP && key < see_max; ++key) {
            const size_t b = (size_t)pages[key / kPage] * a.n_kv_heads + h;
            const uint8_t* v = a.v_pool + (b * kPage + key % kPage) * HD + 4 * half;
#pragma unroll
            for (int d = 0; d < DT; ++d)
#pragma unroll
              for (int g = 0; g < 4; ++g) {
                const uint32_t b = *reinterpret_cast<const uint32_t*>(v + 32 * d + 8 * g);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                  const bool bad = key < see && ((b >> (8 * e)) & 0x7Fu) == 0x7Fu;
                  acc[d][4 * g + e] = bad ? __builtin_nanf("") : acc[d][4 * g + e];
                }
              }
          }
        }
        turn ^= 1;
      }

      const bool whole = step == 0 && stop == steps;
      const int side = step == 0 ? 1 : 0;
      if (!whole) {  // the workers of its first and last steps
        const long long end = pos + ticks - upto, begin = end - steps;
        note(side, sh.team_at(begin), sh.team_at(end - 1), c0, columns, q);
      }
      const float l = sum.of + __shfl_xor(sum.of, 32);
      if (own && whole) {
        f16* dst = a.out + ((size_t)(q.row0 + col / a.group) * a.n_heads + h * a.group +
                            col % a.group) * HD + 4 * half;
#pragma unroll
        for (int d = 0; d < DT; ++d)
#pragma unroll
          for (int g = 0; g < 4; ++g) {
            f16x2 o[2];
#pragma unroll
            for (int e = 0; e < 4; ++e)
              o[e / 2][e % 2] = see > 0 ? (f16)(acc[d][4 * g + e] / l) : (f16)0;
            uint2 v;
            v.x = __builtin_bit_cast(uint32_t, o[0]);
            v.y = __builtin_bit_cast(uint32_t, o[1]);
            *reinterpret_cast<uint2*>(dst + 32 * d + 8 * g) = v;
          }
      } else if (own) {
        const size_t slot = (2 * (size_t)worker + side) * C + c;
        float* dst = a.parts + slot * HD + 4 * half;
#pragma unroll
        for (int d = 0; d < DT; ++d)
#pragma unroll
          for (int g = 0; g < 4; ++g)
            *reinterpret_cast<f32x4*>(dst + 32 * d + 8 * g) =
                f32x4{acc[d][4 * g], acc[d][4 * g + 1], acc[d][4 * g + 2], acc[d][4 * g + 3]};
        if (half == 0) a.parts_ml[slot] = make_float2(m, l);
      }
    }
    tick = 0;
    ++tile;
    while (tile * C >= q.columns && s < a.batch.n_seqs - 1) {
      tile = 0;
      q = same(seq_of(a, ++s));
    }
    if (tile * C >= q.columns) break;
    steps = same(tile_steps<HD, C>(a, q, tile));
  }
}

template <int HD>
int join_launch(const AttentionArgs& a, int columns, hipStream_t stream) {
  if (!a.parts) return LLMK_OK;
  return launch(k_kv8_attention_join<HD>, dim3(a.workers, columns * HD / 1024), dim3(256), 0,
                stream, a, columns);
}

template <int HD, int QT>
int few_launch(AttentionArgs a, hipStream_t stream) {
  const bool two = QT == 1 && a.batch.max_pages <= kShortPages &&
                   (long long)a.batch.n_seqs * a.n_kv_heads >= 2 * kFewWorkers;
  a.workers = two ? 2 * kFewWorkers : kFewWorkers;
  a.teams = a.workers / a.n_kv_heads;
  const int st =
      launch(k_kv8_attention_few<HD, QT>, dim3(a.workers / 4), dim3(256), 0, stream, a);
  return st != LLMK_OK ? st : join_launch<HD>(a, 16 * QT, stream);
}

template <int HD, int W>
int many_launch(AttentionArgs a, hipStream_t stream) {
  a.workers = kManyWorkers<W>;
  a.teams = a.workers / a.n_kv_heads;
  const int st =
      launch(k_kv8_attention_many<HD, W>, dim3(a.workers), dim3(64 * W), 0, stream, a);
  return st != LLMK_OK ? st : join_launch<HD>(a, 32 * W, stream);
}

// Sequences of up to kFewColumns columns go by waves, longer ones by blocks. One launch serves all
// where max_rows, or a single sequence, says that there is one kind; more columns than were
// announced are then several tiles.
template <int HD>
int attention_launch(AttentionArgs a, int max_rows, hipStream_t stream) {
  const long long columns = (long long)max_rows * a.group;
  if (columns <= 16) return few_launch<HD, 1>(a, stream);
  if (columns <= kFewColumns) return few_launch<HD, 2>(a, stream);
  if (a.batch.n_seqs > 1) {
    a.most_columns = kMixedColumns;
    const int st = few_launch<HD, 2>(a, stream);
    if (st != LLMK_OK) return st;
    a.most_columns = 0x7FFFFFFF;
    a.least_columns = kMixedColumns + 1;
  }
  return columns <= kWideColumns || a.n_kv_heads > kManyWorkers<8> ? many_launch<HD, 4>(a, stream)
                                                                   : many_launch<HD, 8>(a, stream);
}

}  // namespace
}  // namespace llmk

using namespace llmk;

extern "C" size_t llmk_kv8_attention_workspace_floats(int head_dim) {
  if (head_dim != 64 && head_dim != 128) return 0;
  return (size_t)kSlotColumns * (head_dim + 2) + 2 * kWorkers * (sizeof(Shared) / 4);
}

extern "C" int llmk_kv8_attention(const uint16_t* q, const uint8_t* k_pool, const float* k_scale,
                                  const uint8_t* v_pool, const float* v_scale,
                                  const int32_t* block_tables, const int32_t* row_starts,
                                  const int32_t* seq_lens, uint16_t* out, float* workspace,
                                  int n_rows, int n_seqs, int max_rows, int max_pages,
                                  int page_size, int n_heads, int n_kv_heads, int head_dim,
                                  void* stream) {
  if (n_rows < 0 || n_seqs < 0 || max_rows < 0 || max_pages <= 0 || n_heads <= 0 ||
      n_kv_heads <= 0 || head_dim <= 0)
    return LLMK_ERR_INVALID_VALUE;
  if (!row_starts && n_rows != n_seqs) return LLMK_ERR_INVALID_VALUE;
  if (page_size != kv8::kPage || (head_dim != 64 && head_dim != 128) || n_heads % n_kv_heads != 0)
    return LLMK_ERR_SHAPE;
  if (n_rows == 0 || n_seqs == 0) return LLMK_OK;
  if (max_rows == 0 || !q || !k_pool || !k_scale || !v_pool || !v_scale || !block_tables ||
      !seq_lens || !out)
    return LLMK_ERR_INVALID_VALUE;
  // a sequence's columns, and positions of a table, are counted in 32 bits
  if ((long long)n_rows * (n_heads / n_kv_heads) > 0x7FFF0000LL || n_heads > 65535 ||
      n_kv_heads > kMostKvHeads || max_pages > 0x7FFF0000 / kv8::kPage)
    return LLMK_ERR_UNSUPPORTED;
  if (!aligned16(q) || !aligned16(k_pool) || !aligned16(v_pool) || !aligned16(out) ||
      !aligned16(workspace))
    return LLMK_ERR_ALIGNMENT;
  AttentionArgs a;
  a.batch = kv8::Batch{block_tables, row_starts, seq_lens, n_rows, n_seqs, max_pages};
  a.q = reinterpret_cast<const f16*>(q);
  a.k_pool = k_pool;
  a.k_scale = k_scale;
  a.v_pool = v_pool;
  a.v_scale = v_scale;
  a.out = reinterpret_cast<f16*>(out);
  a.parts = max_pages > whole_pages(head_dim) ? workspace : nullptr;
  a.parts_ml = reinterpret_cast<float2*>(workspace + (size_t)kSlotColumns * head_dim);
  a.shared = reinterpret_cast<Shared*>(workspace + (size_t)kSlotColumns * (head_dim + 2));
  a.n_heads = n_heads;
  a.n_kv_heads = n_kv_heads;
  a.group = n_heads / n_kv_heads;
  a.workers = a.teams = 0;
  a.least_columns = 0;
  a.most_columns = 0x7FFFFFFF;
  hipStream_t s = static_cast<hipStream_t>(stream);
  return head_dim == 64 ? attention_launch<64>(a, max_rows, s)
                        : attention_launch<128>(a, max_rows, s);
}
