// Low-rank adapters of a batch's sequences beside a shared projection:
//   y[r, :] += scale_a B_a h, h = A_a x[r, :], a the adapter of row r's sequence.
//
// Matrix products over tiles of 16 rows that have the same adapter, so that its weights are read once for them.
// Bound by bytes: A and B of the adapters present, x, and y both ways; a prompt's by y. In two launches:
// k_lora_shrink finds the tiles and computes h, k_lora_expand adds B_a h to y; or in one, k_lora_whole, where a
// block's columns are few enough blocks that each may compute its h again.
//
// Measured (one MI355X, fp16, inputs from HBM; the floor is each byte once at 6 TB/s), us:
//   1 row, rank 16, 2048 -> 2048: 5.1 (< 0.1). One launch: its loads one behind the other.
//   48 sequences of up to 5 rows, 16 adapters of rank 16, 4096 -> 4096|1024|1024: 10.5 (2.2). One launch; every block
//     reads its tile's A and x again, from the L2: 8.9 where all of it is in the last-level cache.
//   256 rows of 100 adapters of ranks up to 64, 8192 -> 2048: 28.7 (12.6), 18 and 10. 61 MB by the first launch at 3.3
//     TB/s: a tile's rows are found (2 us), then two rounds of loads that wait for one another.
//   4 prompts of up to 1001 rows, ranks up to 32, 2048 -> 8192|8192: 42.1 (27.7), 9 and 35. y in place by 16 rows of
//     256 bytes a wave, which alone take 30.
//   3 prompts of 456 rows, rank 128, 8192 -> 11008|11008: 89 (30.6), 40 and 57. A and B from the L2 by every tile, 540
//     MB for the first; two tiles a block halve that, but also the waves a SIMD, and take as long.
//
// Tiles. Sequences are taken 256 at a time (a window); those of a window with the same adapter are a group, in the
// order of their first ones, and a group's rows, in order, are cut into tiles of 16. Every block of the first
// product finds its tile by itself: up to 64 sequences by a wave, whose lanes compare adapters bit by bit; more by
// adapters in a hash table in LDS, whose slots collect the rows and the first member, and counts of tiles summed up
// by those. That takes half a microsecond, or one and a half, beside the loads of ids and starts, which a launch of
// its own would have to wait for too. What a block finds does not depend on the order in which threads reach the
// table. Window w's tiles begin at slot starts[256 w] / 16 + w * (groups + 1), which leaves room for all of them:
// slots without a tile are noted as such.
//
// Between the products h is held in fp32 (the blocks of a tile that share out in_features leave a sum
// each) and given to the matrix instructions as two fp16: h * 2^-e, with 2^e such that the row's largest
// is from 2^14 to 2^15, rounded, and what that lost. That keeps 22 bits relative to the row's largest, and the sum
// is multiplied by scale * 2^e in fp32. So neither large nor small values of h leave fp16's range. Infinities of A and
// B come out as the formula has them (expand_columns).
#include <math.h>

#include "kv8.hpp"
#include "lora_plan.hpp"
#include "overlap.hpp"

namespace llmk {
namespace {

using namespace lora;

typedef float f32x4 __attribute__((ext_vector_type(4)));

constexpr int kHash = 512;
constexpr int kNote = 32;  // ints of a tile's note: adapter (-1: no tile), rank, scale; from 16 on its rows (-1: none)

struct LoraArgs {
  const f16 *x, *a, *b;
  const int *ranks, *ids, *starts;
  const float* scales;
  f16* y;
  int* notes;   // workspace: [slots, kNote]
  f32x4* h;     // [splits, slots, n_parts, steps of 32 ranks, 2, 64]: lane by lane as the second product wants it
  int part_end[kParts], chunk_end[kParts];  // columns, and blocks of k_lora_expand, up to each part's end
  int ldx, ldy, n_parts, n_rows, n_seqs, n_adapters, max_rank, in;
  int slots, splits, groups, windows, steps;
  int turns;      // blocks of k_lora_shrink that share out the products of a tile and split
  int per_block;  // tiles of a block of k_lora_expand; for k_lora_whole, whether a tile's blocks share an XCD
};

__device__ __forceinline__ int first_row(const LoraArgs& g, int s) {
  const int r = g.starts ? g.starts[s] : s;
  return r < 0 ? 0 : r < g.n_rows ? r : g.n_rows;
}

__device__ __forceinline__ int slot_of_window(const LoraArgs& g, int w) {
  return first_row(g, min(w * kWindow, g.n_seqs)) / kRows + w * (g.groups + 1);
}

// The sum of v over the threads in front, of the first 256. part: four ints that no thread still reads.
__device__ __forceinline__ int block_scan(int v, int* part) {
  const int wave = threadIdx.x >> 6, in = wave_scan(v);
  if ((threadIdx.x & 63) == 63 && wave < 4) part[wave] = in;
  lds_barrier();
  int before = 0;
#pragma unroll
  for (int w = 0; w < 3; ++w) before += w < wave ? part[w] : 0;
  return before + in - v;
}

// A value that all lanes have, in a scalar register.
__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }

struct Plan {
  int key[kHash];            // the adapter of a slot of the table, -1: none
  int rows[kHash];           // its rows
  int first[kHash];          // its first member
  int part[2][4];
  int adapter, group, from;  // of the tile: its group's table slot, and its first row among the group's
  int rank;
  float scale;
  int row[kRows];
};

// What a wave writes to its own part of LDS is there for all of its lanes.
__device__ __forceinline__ void wave_sync() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

struct Tile {  // its adapter (-1: there is no tile) and what belongs to that; the rows are in Plan::row
  int adapter, rank;
  float scale;
};

// The members of a tile that have rows of it, one behind the other: lane i's row, of 16. before: a member's first row
// among the tile's.
__device__ __forceinline__ int row_of_tile(uint64_t members, int before, int rows, int r0, int row) {
  const int lane = threadIdx.x & 63;
  for (; members; members &= members - 1) {
    const int from = __builtin_ctzll(members);
    const int i = lane - __builtin_amdgcn_readlane(before, from);
    if (i >= 0 && i < __builtin_amdgcn_readlane(rows, from)) row = __builtin_amdgcn_readlane(r0, from) + i;
  }
  return row;
}

// Finds tile `slot` among 64 sequences at most: every wave by itself, a sequence a lane, without a barrier. All write
// the same rows.
__device__ __forceinline__ Tile find_tile_by_wave(const LoraArgs& g, int slot, Plan& p) {
  const int lane = threadIdx.x & 63;
  int id = -1, r0 = 0, rows = 0, rank = g.max_rank;
  float scale = 1.f;
  if (lane < g.n_seqs) {
    id = g.ids[lane];
    r0 = first_row(g, lane);
    rows = g.starts ? max(first_row(g, lane + 1) - r0, 0) : 1;
    if ((unsigned)id >= (unsigned)g.n_adapters || rows == 0) id = -1;
  }
  if (id >= 0) {
    if (g.ranks) rank = g.ranks[id];
    if (g.scales) scale = g.scales[id];
  }
  uint64_t group = __builtin_amdgcn_ballot_w64(id >= 0);  // the lanes of the same adapter, bit by bit of its number
  const int numbers = g.n_seqs > 1 ? g.n_adapters - 1 : 0;
  for (int bit = 0; numbers >> bit; ++bit) {
    const bool set = id >> bit & 1;
    const uint64_t all = __builtin_amdgcn_ballot_w64(set);
    group &= set ? all : ~all;
  }
  const int leader = id >= 0 ? __builtin_ctzll(group) : lane;
  int total = __builtin_popcountll(group);
  if (g.starts) {
    int* sums = p.rows + (threadIdx.x & ~63);
    sums[lane] = 0;
    wave_sync();
    if (id >= 0) atomicAdd(&sums[leader], rows);
    wave_sync();
    total = sums[lane];
  }
  const bool leads = id >= 0 && leader == lane;
  const int tiles = leads ? (total + kRows - 1) / kRows : 0, upto = wave_scan(tiles);
  const int tile = slot - uniform(first_row(g, 0)) / kRows;
  const uint64_t here = __builtin_amdgcn_ballot_w64(leads && tile >= upto - tiles && tile < upto);
  if (here == 0) {
    if (lane < kRows) p.row[lane] = -1;  // the note's
    wave_sync();
    return {-1, 0, 0.f};
  }
  const int first = __builtin_ctzll(here);
  const bool mine = id >= 0 && leader == first;
  const int from = (tile - __builtin_amdgcn_readlane(upto - tiles, first)) * kRows;
  const int before = wave_scan(mine ? rows : 0) - rows - from;
  const int row = row_of_tile(
      __builtin_amdgcn_ballot_w64(mine && before < kRows && before + rows > 0), before, rows, r0, -1);
  if (lane < kRows) p.row[lane] = row;
  wave_sync();
  return {__builtin_amdgcn_readlane(id, first), min(__builtin_amdgcn_readlane(rank, first), g.max_rank),
          __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, scale), first))};
}

// Finds tile `slot` with 256 threads or more.
__device__ __forceinline__ Tile find_tile(const LoraArgs& g, int slot, Plan& p) {
  // 48 sequences of 16 adapters take 10.4 us so and 11.2 by the table, 8 of 8 9.5 and 10.5 (rank 32)
  if (g.n_seqs <= 64) return find_tile_by_wave(g, slot, p);
  const int tid = threadIdx.x;
  int w = 0;
  for (int hi = g.windows; hi - w > 1;) {  // the last window that begins at or before the slot
    const int mid = (w + hi) / 2;
    if (slot_of_window(g, mid) <= slot) w = mid; else hi = mid;
  }
  const int s = w * kWindow + tid;
  int id = -1, r0 = 0, rows = 0;
  if (tid < kWindow && s < g.n_seqs) {
    id = g.ids[s];
    r0 = first_row(g, s);
    rows = g.starts ? max(first_row(g, s + 1) - r0, 0) : 1;
    if ((unsigned)id >= (unsigned)g.n_adapters || rows == 0) id = -1;
  }
  const int tile = slot - slot_of_window(g, w);
#pragma unroll
  for (int i = tid; i < kHash; i += kWindow) {
    p.key[i] = -1;
    p.rows[i] = 0;
    p.first[i] = kWindow;
  }
  if (tid < kRows) p.row[tid] = -1;
  if (tid == 0) p.adapter = -1;
  lds_barrier();
  // what the first member will note is on its way while the table fills
  int rank = g.max_rank;
  float scale = 1.f;
  int at = -1;
  if (id >= 0) {  // at most kWindow adapters in kHash slots: the search ends
    if (g.ranks) rank = g.ranks[id];
    if (g.scales) scale = g.scales[id];
    at = (int)(((unsigned)id * 2654435761u) >> 23);
    for (;;) {
      const int was = atomicCAS(&p.key[at], -1, id);
      if (was == -1 || was == id) break;
      at = (at + 1) & (kHash - 1);
    }
    atomicAdd(&p.rows[at], rows);
    atomicMin(&p.first[at], tid);
  }
  lds_barrier();
  const bool leads = at >= 0 && p.first[at] == tid;
  const int tiles = leads ? (p.rows[at] + kRows - 1) / kRows : 0;
  const int begin = block_scan(tiles, p.part[0]);
  if (leads && tile >= begin && tile < begin + tiles) {
    p.adapter = id;
    p.group = at;
    p.from = (tile - begin) * kRows;
    p.rank = min(rank, g.max_rank);
    p.scale = scale;
  }
  lds_barrier();
  if (p.adapter < 0) return {-1, 0, 0.f};
  const bool mine = at == p.group;
  const int before = block_scan(mine ? rows : 0, p.part[1]) - p.from;
  // a wave whose members have rows of it writes those
  const uint64_t members =
      __builtin_amdgcn_ballot_w64(mine && before < kRows && before + rows > 0);
  const int row = row_of_tile(members, before, rows, r0, -1);
  if ((tid & 63) < kRows && row >= 0) p.row[tid & 63] = row;
  lds_barrier();
  return {uniform(p.adapter), uniform(p.rank), __builtin_bit_cast(float, uniform(__builtin_bit_cast(int, p.scale)))};
}

// 16 rows of 512 bytes in LDS, in pieces of 16, which lie such that neither a row's 32 pieces nor a piece of
// all rows share banks.
typedef u32x4 Stage[kRows * 32 + 4];  // and four more for 16 numbers behind them
__device__ __forceinline__ int place_of(int row, int piece) { return row * 32 + (piece ^ row); }

__device__ __forceinline__ void put_rows(u32x4* to, const u32x4 (&v)[8], int lane) {
#pragma unroll
  for (int t = 0; t < 8; ++t) to[place_of(2 * t + (lane >> 5), lane & 31)] = v[t];
}
__device__ __forceinline__ void get_rows(const u32x4* from, u32x4 (&v)[8], int n, int q) {
#pragma unroll
  for (int t = 0; t < 8; ++t) v[t] = from[place_of(n, 4 * t + q)];
}

// acc[i] += W_i x for the chunks of in_features that a wave takes: D[rank, row]. A chunk's rows are 512 bytes,
// loaded two an instruction, in whole lines, all of them on their way before the first product waits for one, and
// go through LDS to where the matrix instructions want them (row n, eight numbers from 8 q on in each step of
// 32). Loaded as these want them, 64 bytes of 16 rows an instruction, they take three times as long: 8000
// cycles for 32 instructions of four waves from the L2, not 2400. x: the lane's rows; w: of the lane's first row,
// `rows` behind it clamped. Products `most` and behind are none.
// SOME: of x only the rows that there are, n_x instructions' worth or up to as many again; the others' numbers are what
// LDS holds, and give what nobody reads.
template <int NG, bool SOME>
__device__ __forceinline__ void shrink_chunks(f32x4 (&acc)[NG], const LoraArgs& g, const int (&row)[8],
                                              const f16* const (&w)[NG], const int (&left)[NG], int most,
                                              int chunk, int step, u32x4* stage, int lane, int n_x = 8) {
  const int n = lane & 15, q = lane >> 4, r = lane >> 5, at = 8 * (lane & 31), in = g.in;
  const auto there = [&](int t) { return !SOME || t == 0 || n_x > (t == 1 ? 1 : t < 4 ? 2 : 4); };
  for (int c = chunk; c * kChunk < in; c += step) {
    const int k0 = c * kChunk + at, k = min(k0, in - 8);  // past in_features: loaded, and cleared below
    u32x4 xr[8], wr[NG][8], xf[8], wf[8];
#pragma unroll
    for (int t = 0; t < 8; ++t)
      if (there(t)) xr[t] = ld16(g.x + (size_t)row[t] * g.ldx + k);
#pragma unroll
    for (int i = 0; i < NG; ++i)
      if (i < most)
#pragma unroll
        for (int t = 0; t < 8; ++t) wr[i][t] = ld16(w[i] + (uint32_t)(min(2 * t + r, left[i]) * in + k));
    if ((c + 1) * kChunk > in) {
#pragma unroll
      for (int t = 0; t < 8; ++t) xr[t] = k0 < in ? xr[t] : u32x4{0, 0, 0, 0};
#pragma unroll
      for (int i = 0; i < NG; ++i)
#pragma unroll
        for (int t = 0; t < 8; ++t) wr[i][t] = k0 < in ? wr[i][t] : u32x4{0, 0, 0, 0};
    }
#pragma unroll
    for (int t = 0; t < 8; ++t)
      if (there(t)) stage[place_of(2 * t + r, lane & 31)] = xr[t];
    wave_sync();
    get_rows(stage, xf, n, q);
    wave_sync();
#pragma unroll
    for (int i = 0; i < NG; ++i) {
      if (i >= most) break;
      put_rows(stage, wr[i], lane);
      wave_sync();
      get_rows(stage, wf, n, q);
      __builtin_amdgcn_sched_barrier(0);  // all reads in front of the first product
#pragma unroll
      for (int t = 0; t < 8; ++t)
        acc[i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(as_h8(wf[t]), as_h8(xf[t]), acc[i], 0, 0, 0);
      wave_sync();
    }
  }
}

// The rows of x that a lane loads; for one that is none, one that is: it gives what nobody reads.
__device__ __forceinline__ void rows_of_x(const Plan& p, int (&row)[8], int lane) {
#pragma unroll
  for (int t = 0; t < 8; ++t) {
    const int r = p.row[2 * t + (lane >> 5)];
    row[t] = r >= 0 ? r : p.row[0];
  }
}

// h of a tile: D[rank, row] = A[rank, k] x[row, k], by waves that take 256 of in_features at a time, NG products of 16
// ranks side by side. Blocks share out a tile's products (turns) and its in_features (splits), as shape_of says.
template <int NG>
__global__ void __launch_bounds__(256, NG == 3 ? 2 : 3) k_lora_shrink(const LoraArgs g) {
  __shared__ Plan p;
  __shared__ Stage stage[4];
  const int slot = blockIdx.x / (g.splits * g.turns), rest = blockIdx.x - slot * g.splits * g.turns;
  const int split = rest / g.turns, turn = rest - split * g.turns;
  const int wave = uniform(threadIdx.x >> 6), lane = threadIdx.x & 63, n = lane & 15, q = lane >> 4;
  const Tile tile = find_tile(g, slot, p);
  const int a = tile.adapter, rank = tile.rank;
  if (rest == 0) {
    int* note = g.notes + (size_t)slot * kNote;
    if (threadIdx.x == 0) {
      note[0] = a;
      note[1] = rank;
      note[2] = __builtin_bit_cast(int, tile.scale);
    }
    if (threadIdx.x < kRows) note[kRows + threadIdx.x] = p.row[threadIdx.x];
  }
  if (a < 0 || rank <= 0) return;
  const int per_part = (rank + 15) / 16, all = g.n_parts * per_part;
  int xrow[8];
  rows_of_x(p, xrow, lane);
  f32x4* out = g.h + ((size_t)split * g.slots + slot) * g.n_parts * g.steps * 128;
  for (int g0 = turn * NG; g0 < all; g0 += g.turns * NG) {
    f32x4 acc[NG];
    const f16* w[NG];
    int left[NG];
#pragma unroll
    for (int i = 0; i < NG; ++i) {
      acc[i] = f32x4{0.f, 0.f, 0.f, 0.f};
      const int gi = min(g0 + i, all - 1), part = gi / per_part, j = (gi - part * per_part) * 16;
      w[i] = g.a + (((size_t)a * g.n_parts + part) * g.max_rank + j) * g.in;
      left[i] = rank - 1 - j;
    }
    if (g0 >= g.turns * NG) lds_barrier();  // behind what is read of the last ones' sums
    shrink_chunks<NG, false>(acc, g, xrow, w, left, all - g0, split * 4 + wave, 4 * g.splits, stage[wave], lane);
    // the four waves' sums
#pragma unroll
    for (int i = 0; i < NG; ++i) stage[wave][i * 64 + lane] = __builtin_bit_cast(u32x4, acc[i]);
    lds_barrier();
    if (wave < NG && g0 + wave < all) {  // wave i adds product i's
      f32x4 v[4];
#pragma unroll
      for (int m = 0; m < 4; ++m) v[m] = __builtin_bit_cast(f32x4, stage[m][wave * 64 + lane]);
      // ranks 4 q on of 16: numbers 4 (q & 1) on of the eight that lane (n, 2 (i & 1) + q / 2) has of step i / 2
      const int part = (g0 + wave) / per_part, i = g0 + wave - part * per_part;
      out[(((size_t)part * g.steps + i / 2) * 2 + (q & 1)) * 64 + (2 * (i & 1) + (q >> 1)) * 16 + n] =
          (v[0] + v[1]) + (v[2] + v[3]);
    }
  }
}

// B's rows for the products of a wave, in steps of 32 ranks. The columns are taken 32 at a time by two products,
// whose rows of B are chosen such that a lane gets eight columns side by side.
template <int KS, int TILES>
__device__ __forceinline__ void load_b(u32x4 (&bf)[TILES][KS], const f16* b, int c0, int end, int max_rank,
                                       int rank, int n, int q) {
#pragma unroll
  for (int t = 0; t < TILES; ++t) {
    const int c = min(c0 + 32 * (t / 2) + 8 * (n / 4) + 4 * (t & 1) + n % 4, end - 1);
#pragma unroll
    for (int s = 0; s < KS; ++s)
      bf[t][s] = 32 * s + 8 * q < rank ? ld16(b + (size_t)c * max_rank + 32 * s + 8 * q) : u32x4{0, 0, 0, 0};
  }
}
// What lies past the rank is not read as numbers.
template <int KS, int TILES>
__device__ __forceinline__ void cut_b(u32x4 (&bf)[TILES][KS], int rank, int q) {
  if (rank % 8 == 0) return;
#pragma unroll
  for (int t = 0; t < TILES; ++t)
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      f16x8 v = as_h8(bf[t][s]);
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = 32 * s + 8 * q + e < rank ? v[e] : (f16)0;
      bf[t][s] = as_u4(v);
    }
}

// 2^e for a row whose largest magnitude is `most`: that times 2^-e (*down) is from 2^14 to 2^15.
__device__ __forceinline__ float power_of(float most, float* down) {
  int e = (int)(__builtin_bit_cast(uint32_t, most) >> 23) - 127 - 14;
  e = e < -100 ? -100 : e;
  *down = kv8::exp2_int(-e);
  return kv8::exp2_int(e);
}
// Eight numbers times 2^-e as two fp16 each.
__device__ __forceinline__ void two_halves(const float (&v)[8], float down, f16x8& hi, f16x8& lo) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float u = v[i] * down;
    hi[i] = (f16)u;
    lo[i] = __builtin_fabsf(u) < INFINITY ? (f16)(u - (float)hi[i]) : (f16)0;
  }
}

// A lane's h (row n, ranks 32 s + 8 q on) as two fp16 each; returns the 2^e that they are to be multiplied by.
template <int KS>
__device__ __forceinline__ float split_h(const float (&v)[KS][8], f16x8 (&hi)[KS], f16x8 (&lo)[KS]) {
  float most = 0.f;
#pragma unroll
  for (int s = 0; s < KS; ++s)
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float mag = __builtin_fabsf(v[s][e]);
      most = mag < INFINITY ? __builtin_fmaxf(most, mag) : most;
    }
  most = __builtin_fmaxf(most, __shfl_xor(most, 16));
  most = __builtin_fmaxf(most, __shfl_xor(most, 32));
  float down;
  const float up = power_of(most, &down);
#pragma unroll
  for (int s = 0; s < KS; ++s) two_halves(v[s], down, hi[s], lo[s]);
  return up;
}

// v with its infinities and NaN as 0.
__device__ __forceinline__ u32x4 finite_of(u32x4 v) {
  f16x8 x = as_h8(v);
#pragma unroll
  for (int e = 0; e < 8; ++e) x[e] = __builtin_fabsf((float)x[e]) < INFINITY ? x[e] : (f16)0;
  return as_u4(x);
}

// B h of a wave's 16 rows and 16 * TILES columns: row n, columns 32 t + 8 q on of each pair of products, into LDS
// (in pieces of 16 bytes as above); and what the row's are to be multiplied by, behind them. Where a sum is no number
// it is made again, the lower halves of h by B's finite numbers alone: an infinity of B times a lower half, which may be
// 0 or of the other sign, is NaN, and the product's is an infinity. h_of: the halves of h once more.
template <int KS, int TILES, typename H>
__device__ __forceinline__ void expand_columns(const u32x4 (&bf)[TILES][KS], const f16x8 (&hi)[KS],
                                               const f16x8 (&lo)[KS], float by, u32x4* to, int n, int q, H h_of) {
  const auto place = [&](int t) { return n * 4 * TILES + ((8 * (t / 2) + 2 * q + (t & 1)) ^ (n & (4 * TILES - 1))); };
  bool none = false;
#pragma unroll
  for (int t = 0; t < TILES; ++t) {
    f32x4 d = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      d = __builtin_amdgcn_mfma_f32_16x16x32_f16(as_h8(bf[t][s]), hi[s], d, 0, 0, 0);
      d = __builtin_amdgcn_mfma_f32_16x16x32_f16(as_h8(bf[t][s]), lo[s], d, 0, 0, 0);
    }
    to[place(t)] = __builtin_bit_cast(u32x4, d);
    const float sum = (d[0] + d[1]) + (d[2] + d[3]);
    none |= sum != sum;
  }
  if (__builtin_amdgcn_ballot_w64(none)) {
    wave_sync();
#pragma unroll
    for (int t = 0; t < TILES; ++t) {
      f32x4 d = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int s = 0; s < KS; ++s) {
        f16x8 high, low;
        __builtin_amdgcn_sched_barrier(0);  // one step's at a time
        h_of(s, high, low);
        d = __builtin_amdgcn_mfma_f32_16x16x32_f16(as_h8(bf[t][s]), high, d, 0, 0, 0);
        d = __builtin_amdgcn_mfma_f32_16x16x32_f16(as_h8(finite_of(bf[t][s])), low, d, 0, 0, 0);
      }
      to[place(t)] = __builtin_bit_cast(u32x4, d);
    }
  }
  if (q == 0) reinterpret_cast<float*>(to + kRows * 4 * TILES)[n] = by;
}

// A wave's y: 2 * TILES lanes a row, eight columns each, so that accesses are of whole lines. row(t) is the
// lane's t-th row among the 16; `inside`: whether its columns are the part's.
template <int TILES>
__device__ __forceinline__ int y_row(int t, int lane) { return t * (32 / TILES) + lane / (2 * TILES); }

// Whether all of the wave's accesses are: most tiles have 16 rows and most waves only columns of the part.
template <int TILES>
__device__ __forceinline__ bool all_of(f16* const (&y)[TILES / 2]) {
  bool all = true;
#pragma unroll
  for (int t = 0; t < TILES / 2; ++t) all &= y[t] != nullptr;
  return __builtin_amdgcn_ballot_w64(all) == ~0ull;
}

template <int TILES>
__device__ __forceinline__ void load_y(u32x4 (&old)[TILES / 2], f16* const (&y)[TILES / 2], bool all) {
  if (all) {
#pragma unroll
    for (int t = 0; t < TILES / 2; ++t) old[t] = ld16_stream(y[t]);
  } else {
#pragma unroll
    for (int t = 0; t < TILES / 2; ++t)
      if (y[t]) old[t] = ld16_stream(y[t]);
  }
}

template <int TILES>
__device__ __forceinline__ void add_to_y(u32x4 (&old)[TILES / 2], f16* const (&y)[TILES / 2], bool all,
                                         const u32x4* from, int lane) {
#pragma unroll
  for (int t = 0; t < TILES / 2; ++t) {
    const int r = y_row<TILES>(t, lane), piece = 2 * (lane % (2 * TILES)), flip = r & (4 * TILES - 1);
    const f32x4 u = __builtin_bit_cast(f32x4, from[r * 4 * TILES + (piece ^ flip)]);
    const f32x4 w = __builtin_bit_cast(f32x4, from[r * 4 * TILES + ((piece + 1) ^ flip)]);
    const float by = reinterpret_cast<const float*>(from + kRows * 4 * TILES)[r];
    f16x8 v = as_h8(old[t]);
#pragma unroll
    for (int e = 0; e < 4; ++e) {  // an instruction each: product and sum in fp32, one rounding
      v[e] = (f16)__builtin_fmaf(u[e], by, (float)v[e]);
      v[e + 4] = (f16)__builtin_fmaf(w[e], by, (float)v[e + 4]);
    }
    old[t] = as_u4(v);
  }
  if (all) {
#pragma unroll
    for (int t = 0; t < TILES / 2; ++t) st16_stream(y[t], old[t]);
  } else {
#pragma unroll
    for (int t = 0; t < TILES / 2; ++t)
      if (y[t]) st16_stream(y[t], old[t]);
  }
}

// The part that a block's columns lie in, and the block's place in it.
__device__ __forceinline__ int part_of(const LoraArgs& g, int chunk, int* place) {
  int part = 0;
  while (chunk >= g.chunk_end[part]) ++part;
  *place = chunk - (part ? g.chunk_end[part - 1] : 0);
  return part;
}

// y of a tile's rows: D[column, row] = B[column, j] h[row, j]. Waves work by themselves; those of a block take
// columns side by side, so that h comes from the first-level cache but once. A wave keeps its columns of B while
// its tiles, `per_block` in a row, have the same adapter. MANY: more than two splits, whose sums the block's waves
// share out.
template <int KS, bool MANY>
__global__ void __launch_bounds__(256, KS == 1 ? 3 : 2) k_lora_expand(const LoraArgs g) {
  constexpr int TILES = 8;
  __shared__ u32x4 stage[4][kRows * 4 * TILES + 4];
  const int wave = uniform(threadIdx.x >> 6), lane = threadIdx.x & 63, n = lane & 15, q = lane >> 4;
  int place;
  const int chunks = g.chunk_end[g.n_parts - 1];
  const int part = part_of(g, blockIdx.x % chunks, &place);
  const int end = g.part_end[part], out = g.part_end[g.n_parts - 1];
  const int c0 = (part ? g.part_end[part - 1] : 0) + (place * 4 + wave) * 16 * TILES;
  if (!MANY && c0 >= end) return;
  const int column = c0 + 8 * (lane % (2 * TILES));
  __shared__ f32x4 shared_h[MANY ? 4 : 1][KS][2][64];
  u32x4 bf[TILES][KS];
  int loaded = -1;
  const int first = blockIdx.x / chunks * g.per_block, behind = min(first + g.per_block, g.slots);
  for (int slot = first; slot < behind; ++slot) {
    const int* note = g.notes + (size_t)slot * kNote;
    const int a = note[0], rank = note[1];
    const float scale = __builtin_bit_cast(float, note[2]);
    int row[TILES / 2];
#pragma unroll
    for (int t = 0; t < TILES / 2; ++t) row[t] = note[kRows + y_row<TILES>(t, lane)];
    if ((unsigned)a >= (unsigned)g.n_adapters || rank <= 0 || rank > g.max_rank) continue;
    // all that the note leads to is on its way before the first of it is waited for: h, then y and B
    const f32x4* from = g.h + ((size_t)slot * g.n_parts + part) * g.steps * 128 + lane;
    const auto load_split = [&](f32x4 (&v)[KS][2], int split) {
      const f32x4* u = from + (size_t)split * g.slots * g.n_parts * g.steps * 128;
#pragma unroll
      for (int s = 0; s < KS; ++s)  // steps behind the last: its numbers, which rank cuts off
#pragma unroll
        for (int f = 0; f < 2; ++f) v[s][f] = u[(min(s, g.steps - 1) * 2 + f) * 64];
    };
    // the splits' sums: up to two by the wave itself, more by the block's waves, two each, through LDS
    f32x4 u[KS][2], w[KS][2];
    const int one = MANY ? wave : 0, two = MANY ? wave + 4 : 1;
    if (one < g.splits) load_split(u, one);
    if (two < g.splits) load_split(w, two);
    f16* y[TILES / 2];
    u32x4 old[TILES / 2];
#pragma unroll
    for (int t = 0; t < TILES / 2; ++t)
      y[t] = (unsigned)row[t] < (unsigned)g.n_rows && column < end ? g.y + (size_t)row[t] * g.ldy + column
                                                                   : nullptr;
    const bool all = all_of<TILES>(y);
    load_y<TILES>(old, y, all);
    const bool fresh = a != loaded;
    if (fresh) {
      loaded = a;
      load_b<KS, TILES>(bf, g.b + (size_t)a * out * g.max_rank, c0, end, g.max_rank, rank, n, q);
    }
    if (one < g.splits && two < g.splits)
#pragma unroll
      for (int s = 0; s < KS; ++s)
#pragma unroll
        for (int f = 0; f < 2; ++f) u[s][f] += w[s][f];
    if (MANY) {
      if (slot > first) lds_barrier();  // behind what the waves read of the last tile's
#pragma unroll
      for (int s = 0; s < KS; ++s)
#pragma unroll
        for (int f = 0; f < 2; ++f) shared_h[wave][s][f][lane] = u[s][f];
      lds_barrier();
#pragma unroll
      for (int s = 0; s < KS; ++s)
#pragma unroll
        for (int f = 0; f < 2; ++f) {
          f32x4 v[4];
#pragma unroll
          for (int m = 0; m < 4; ++m)
            if (m < g.splits) v[m] = shared_h[m][s][f][lane];
          u[s][f] = v[0];
#pragma unroll
          for (int m = 1; m < 4; ++m)
            if (m < g.splits) u[s][f] += v[m];
        }
    }
    float h[KS][8];
#pragma unroll
    for (int s = 0; s < KS; ++s)
#pragma unroll
      for (int e = 0; e < 8; ++e) h[s][e] = 32 * s + 8 * q + e < rank ? u[s][e / 4][e % 4] : 0.f;
    if (fresh) cut_b<KS, TILES>(bf, rank, q);
    f16x8 hi[KS], lo[KS];
    const float by = scale * split_h<KS>(h, hi, lo);
    const auto of_registers = [&](int s, f16x8& high, f16x8& low) { high = hi[s], low = lo[s]; };
    wave_sync();
    expand_columns<KS, TILES>(bf, hi, lo, by, stage[wave], n, q, of_registers);
    wave_sync();
    add_to_y<TILES>(old, y, all, stage[wave], lane);
  }
}

// The same for more than 64 ranks: a block's waves share out the steps of 32 ranks, add up their splits and make them
// the two fp16 once for all. 3 prompts of 456 rows and rank 128 on 11008|11008 columns take 57 us, and 112 with h made
// by every wave for itself and half the columns.
template <int KS>
__global__ void __launch_bounds__(256, 2) k_lora_expand_high(const LoraArgs g) {
  constexpr int TILES = 32 / KS, MINE = KS / 4, AT = KS == 4 ? 4 : 1;  // AT: splits at a time, as registers allow
  __shared__ u32x4 stage[4][kRows * 4 * TILES + 4];
  __shared__ u32x4 pair[KS][2][64];
  __shared__ float top[KS][kRows];
  const int wave = uniform(threadIdx.x >> 6), lane = threadIdx.x & 63, n = lane & 15, q = lane >> 4;
  int place;
  const int chunks = g.chunk_end[g.n_parts - 1];
  const int part = part_of(g, blockIdx.x % chunks, &place);
  const int end = g.part_end[part], out = g.part_end[g.n_parts - 1];
  const int c0 = (part ? g.part_end[part - 1] : 0) + (place * 4 + wave) * 16 * TILES;
  const int column = c0 + 8 * (lane % (2 * TILES));
  u32x4 bf[TILES][KS];
  int loaded = -1;
  const int first = blockIdx.x / chunks * g.per_block, behind = min(first + g.per_block, g.slots);
  for (int slot = first; slot < behind; ++slot) {
    const int* note = g.notes + (size_t)slot * kNote;
    const int a = note[0], rank = note[1];
    const float scale = __builtin_bit_cast(float, note[2]);
    if ((unsigned)a >= (unsigned)g.n_adapters || rank <= 0 || rank > g.max_rank) continue;
    f16* y[TILES / 2];
    u32x4 old[TILES / 2];
#pragma unroll
    for (int t = 0; t < TILES / 2; ++t) {
      const int row = note[kRows + y_row<TILES>(t, lane)];
      y[t] = (unsigned)row < (unsigned)g.n_rows && column < end ? g.y + (size_t)row * g.ldy + column : nullptr;
    }
    // as above: h of the wave's steps, then y and B; with 256 ranks' B, h is out of the registers first
    const f32x4* from = g.h + ((size_t)slot * g.n_parts + part) * g.steps * 128 + lane;
    f32x4 sum[MINE][AT][2];
    const auto load_splits = [&](int d0) {
#pragma unroll
      for (int m = 0; m < MINE; ++m)
#pragma unroll
        for (int k = 0; k < AT; ++k) {
          const f32x4* u = from + (size_t)min(d0 + k, g.splits - 1) * g.slots * g.n_parts * g.steps * 128 +
                           min(wave + 4 * m, g.steps - 1) * 128;
          sum[m][k][0] = u[0];
          sum[m][k][1] = u[64];
        }
    };
    const bool all = all_of<TILES>(y), fresh = a != loaded;
    const auto load_y_and_b = [&] {
      load_y<TILES>(old, y, all);
      if (fresh) load_b<KS, TILES>(bf, g.b + (size_t)a * out * g.max_rank, c0, end, g.max_rank, rank, n, q);
      loaded = a;
    };
    load_splits(0);
    if (KS == 4) load_y_and_b();
    float h[MINE][8];
#pragma unroll
    for (int m = 0; m < MINE; ++m)
#pragma unroll
      for (int e = 0; e < 8; ++e) h[m][e] = 0.f;
    for (int d0 = 0; d0 < g.splits; d0 += AT) {
      if (d0 > 0) load_splits(d0);
#pragma unroll
      for (int m = 0; m < MINE; ++m)
#pragma unroll
        for (int k = 0; k < AT; ++k)
#pragma unroll
          for (int e = 0; e < 8; ++e) h[m][e] += d0 + k < g.splits ? sum[m][k][e / 4][e % 4] : 0.f;
    }
#pragma unroll
    for (int m = 0; m < MINE; ++m) {
      const int s = wave + 4 * m;
      float most = 0.f;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        h[m][e] = 32 * s + 8 * q + e < rank ? h[m][e] : 0.f;
        const float mag = __builtin_fabsf(h[m][e]);
        most = mag < INFINITY ? __builtin_fmaxf(most, mag) : most;
      }
      most = __builtin_fmaxf(most, __shfl_xor(most, 16));
      most = __builtin_fmaxf(most, __shfl_xor(most, 32));
      if (q == 0) top[s][n] = most;
    }
    if (KS == 8) load_y_and_b();
    if (fresh) cut_b<KS, TILES>(bf, rank, q);
    lds_barrier();
    float most = 0.f;
#pragma unroll
    for (int s = 0; s < KS; ++s) most = __builtin_fmaxf(most, top[s][n]);
    float down;
    const float up = power_of(most, &down);
#pragma unroll
    for (int m = 0; m < MINE; ++m) {
      f16x8 hi, lo;
      two_halves(h[m], down, hi, lo);
      pair[wave + 4 * m][0][lane] = as_u4(hi);
      pair[wave + 4 * m][1][lane] = as_u4(lo);
    }
    lds_barrier();
    f16x8 hi[KS], lo[KS];
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      hi[s] = as_h8(pair[s][0][lane]);
      lo[s] = as_h8(pair[s][1][lane]);
    }
    wave_sync();
    expand_columns<KS, TILES>(bf, hi, lo, scale * up, stage[wave], n, q, [&](int s, f16x8& high, f16x8& low) {
      high = as_h8(pair[s][0][lane]);  // held in registers since the first time, they would not fit
      low = as_h8(pair[s][1][lane]);
    });
    wave_sync();
    add_to_y<TILES>(old, y, all, stage[wave], lane);
  }
}

// Both products of a tile and a block's columns in one launch: every block computes the h of its part again.
template <int TILES, int NG>
__global__ void __launch_bounds__(64 * kWaves, 1) k_lora_whole(const LoraArgs g) {
  constexpr int KS = 1;
  __shared__ Plan p;
  __shared__ Stage stage[kWaves];
  // a tile's blocks share an XCD, whose L2 then reads its weights once, unless few tiles would leave most CUs idle
  // (one tile's 64 blocks 8.7 us, and 4.9 for 4)
  const int chunks = g.chunk_end[g.n_parts - 1], turn = g.per_block ? blockIdx.x / 8 : blockIdx.x;
  const int slot = g.per_block ? blockIdx.x % 8 + turn / chunks * 8 : turn / chunks;
  if (slot >= g.slots) return;
  const int wave = uniform(threadIdx.x >> 6), lane = threadIdx.x & 63, n = lane & 15, q = lane >> 4;
  const Tile tile = find_tile(g, slot, p);
  const int a = tile.adapter, rank = tile.rank;
  if (a < 0 || rank <= 0) return;
  int place;
  const int part = part_of(g, turn % chunks, &place);
  const int end = g.part_end[part], out = g.part_end[g.n_parts - 1];
  const int c0 = (part ? g.part_end[part - 1] : 0) + (place * kWaves + wave) * 16 * TILES;
  const int column = c0 + 8 * (lane % (2 * TILES));
  int xrow[8];
  rows_of_x(p, xrow, lane);
  // what the second product needs is loaded in front of the first one
  f16* y[TILES / 2];
  u32x4 old[TILES / 2], bf[TILES][KS];
#pragma unroll
  for (int t = 0; t < TILES / 2; ++t) {
    const int row = p.row[y_row<TILES>(t, lane)];
    y[t] = row >= 0 && column < end ? g.y + (size_t)row * g.ldy + column : nullptr;
  }
  const bool all = all_of<TILES>(y);
  load_y<TILES>(old, y, all);
  load_b<KS, TILES>(bf, g.b + (size_t)a * out * g.max_rank, c0, end, g.max_rank, rank, n, q);
  f32x4 acc[NG];
  const f16* w[NG];
  int left[NG];
#pragma unroll
  for (int i = 0; i < NG; ++i) {
    acc[i] = f32x4{0.f, 0.f, 0.f, 0.f};
    w[i] = g.a + (((size_t)a * g.n_parts + part) * g.max_rank + 16 * i) * g.in;
    left[i] = rank - 1 - 16 * i;
  }
  // Tiles of single tokens have few rows: with one product of 16 ranks they take 5.1 us and not 5.4 on 2048
  // in_features, 5.9 and 6.7 on 4096, tiles of 16 rows as long as before; with two, which leave fewer registers, 12.3
  // and 11.4.
  const int n_x = (__builtin_popcountll(__builtin_amdgcn_ballot_w64(lane < kRows && p.row[lane % kRows] >= 0)) + 1) / 2;
  const int has = p.row[n] >= 0 ? rank : 0;  // the values of a row that is none may be anything
  shrink_chunks<NG, NG == 1>(acc, g, xrow, w, left, (rank + 15) / 16, wave, kWaves, stage[wave], lane, n_x);
#pragma unroll
  for (int i = 0; i < NG; ++i) stage[wave][i * 64 + lane] = __builtin_bit_cast(u32x4, acc[i]);
  lds_barrier();
  float h[KS][8];
#pragma unroll
  for (int s = 0; s < KS; ++s)
#pragma unroll
    for (int f = 0; f < 2; ++f) {
      const int at = (NG == 1 ? 0 : q >> 1) * 64 + (q & 1) * 32 + f * 16 + n;  // NG 1: the ranks past 16 are cut
      f32x4 v[kWaves];
#pragma unroll
      for (int m = 0; m < kWaves; ++m) v[m] = __builtin_bit_cast(f32x4, stage[m][at]);
#pragma unroll
      for (int d = kWaves / 2; d > 0; d /= 2)
#pragma unroll
        for (int m = 0; m < d; ++m) v[m] += v[m + d];
#pragma unroll
      for (int e = 0; e < 4; ++e) h[s][4 * f + e] = 32 * s + 8 * q + 4 * f + e < has ? v[0][e] : 0.f;
    }
  cut_b<KS, TILES>(bf, rank, q);
  f16x8 hi[KS], lo[KS];
  const float by = tile.scale * split_h<KS>(h, hi, lo);
  const auto of_registers = [&](int s, f16x8& high, f16x8& low) { high = hi[s], low = lo[s]; };
  lds_barrier();  // the other waves have read what this one puts its columns over
  expand_columns<KS, TILES>(bf, hi, lo, by, stage[wave], n, q, of_registers);
  wave_sync();
  add_to_y<TILES>(old, y, all, stage[wave], lane);
}

// Elements of an array of so many by so many by .., which a call may name more of than any memory holds.
long long elements(double a, double b, double c = 1, double d = 1) { return (long long)fmin(a * b * c * d, 1e18); }

}  // namespace
}  // namespace llmk

using namespace llmk;

extern "C" size_t llmk_lora_add_workspace_floats(int n_rows, int n_seqs, int n_adapters, int max_rank,
                                                 int in_features, int n_parts) {
  if (n_rows <= 0 || n_seqs <= 0 || n_adapters <= 0 || max_rank <= 0 || in_features <= 0 ||
      n_parts <= 0)
    return 0;
  if (!within_limits(n_rows, n_seqs, max_rank, in_features) || n_parts > kParts) return 0;  // nor is a call
  const Shape s = shape_of(n_rows, n_seqs, n_adapters, in_features, n_parts * ((max_rank + 15) / 16));
  return (size_t)s.slots * (kNote + (size_t)s.splits * n_parts * ((max_rank + 31) / 32) * 512);
}

extern "C" int llmk_lora_add(const uint16_t* x, int ldx, const uint16_t* a, const uint16_t* b,
                             const int32_t* ranks, const float* scales, const int32_t* adapter_ids,
                             const int32_t* row_starts, uint16_t* y, int ldy,
                             const int32_t* part_ends, int n_parts, float* workspace, int n_rows,
                             int n_seqs, int n_adapters, int max_rank, int in_features,
                             void* stream) {
  if (n_rows < 0 || n_seqs < 0 || n_adapters < 0 || max_rank <= 0 || in_features <= 0 ||
      n_parts < 1 || n_parts > kParts || !part_ends || (!row_starts && n_rows != n_seqs))
    return LLMK_ERR_INVALID_VALUE;
  LoraArgs g{};
  for (int p = 0; p < n_parts; ++p) {
    const int begin = p ? part_ends[p - 1] : 0;
    if (part_ends[p] <= begin) return LLMK_ERR_INVALID_VALUE;
    if (part_ends[p] % 8) return LLMK_ERR_SHAPE;
    g.part_end[p] = part_ends[p];
  }
  if (in_features % 8 || max_rank % 8 || ldx % 8 || ldy % 8 || ldx < in_features ||
      ldy < part_ends[n_parts - 1])
    return LLMK_ERR_SHAPE;
  const auto chunks_of = [&](int columns) {  // blocks up to each part's end
    for (int p = 0; p < n_parts; ++p)
      g.chunk_end[p] = (p ? g.chunk_end[p - 1] : 0) + over(part_ends[p] - (p ? part_ends[p - 1] : 0), columns);
    return g.chunk_end[n_parts - 1];
  };
  if (!within_limits(n_rows, n_seqs, max_rank, in_features) || chunks_of(max_rank <= 128 ? 512 : 256) > 65535)
    return LLMK_ERR_UNSUPPORTED;
  if (n_rows == 0 || n_seqs == 0 || n_adapters == 0) return LLMK_OK;
  if (!x || !a || !b || !adapter_ids || !y || !workspace) return LLMK_ERR_INVALID_VALUE;
  if (!aligned16(x) || !aligned16(a) || !aligned16(b) || !aligned16(y) || !aligned16(workspace))
    return LLMK_ERR_ALIGNMENT;
  {  // what is written, and what else there is
    const long long out = part_ends[n_parts - 1];
    const Rows written[] = {
        rows_of(y, n_rows, ldy, out),
        bytes_of(workspace, 4 * llmk_lora_add_workspace_floats(n_rows, n_seqs, n_adapters, max_rank, in_features, n_parts))};
    const auto array = [](const void* p, long long n) { return rows_of(p, 1, 0, n); };  // n elements of 2 bytes
    const Rows others[] = {rows_of(x, n_rows, ldx, in_features),
                           array(a, elements(n_adapters, n_parts, max_rank, in_features)),
                           array(b, elements(n_adapters, out, max_rank)),
                           array(ranks, 2LL * n_adapters),
                           array(scales, 2LL * n_adapters),
                           array(adapter_ids, 2LL * n_seqs),
                           array(row_starts, 2LL * n_seqs + 2)};
    if (overlap(written[0], written[1])) return LLMK_ERR_INVALID_VALUE;
    for (const Rows& w : written)
      for (const Rows& o : others)
        if (overlap(w, o)) return LLMK_ERR_INVALID_VALUE;
  }
  const int per_part = (max_rank + 15) / 16;
  const Shape s = shape_of(n_rows, n_seqs, n_adapters, in_features, n_parts * per_part);
  const Launches l = launches_of(s, n_rows, n_seqs, n_adapters, max_rank, in_features, part_ends, n_parts);
  g.x = reinterpret_cast<const f16*>(x);
  g.a = reinterpret_cast<const f16*>(a);
  g.b = reinterpret_cast<const f16*>(b);
  g.ranks = ranks;
  g.ids = adapter_ids;
  g.starts = row_starts;
  g.scales = scales;
  g.y = reinterpret_cast<f16*>(y);
  g.notes = reinterpret_cast<int*>(workspace);
  g.h = reinterpret_cast<f32x4*>(workspace + (size_t)s.slots * kNote);
  g.ldx = ldx;
  g.ldy = ldy;
  g.n_parts = n_parts;
  g.n_rows = n_rows;
  g.n_seqs = n_seqs;
  g.n_adapters = n_adapters;
  g.max_rank = max_rank;
  g.in = in_features;
  g.slots = s.slots;
  g.steps = (max_rank + 31) / 32;
  g.splits = s.splits;
  g.groups = s.groups;
  g.windows = s.windows;
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (l.one) {
    g.per_block = l.together;
    chunks_of(16 * kWaves * l.tiles);
    return launch(per_part == 1 ? (l.tiles == 2   ? k_lora_whole<2, 1>
                                   : l.tiles == 4 ? k_lora_whole<4, 1>
                                                  : k_lora_whole<8, 1>)
                                : (l.tiles == 2   ? k_lora_whole<2, 2>
                                   : l.tiles == 4 ? k_lora_whole<4, 2>
                                                  : k_lora_whole<8, 2>),
                  dim3((unsigned)l.grid), dim3(64 * kWaves), 0, st, g);
  }
  g.per_block = l.per_block;
  g.turns = s.turns;
  const int status = launch(s.at_once == 1   ? k_lora_shrink<1>
                            : s.at_once == 3 ? k_lora_shrink<3>
                                             : k_lora_shrink<2>,
                            dim3((unsigned)l.grid), dim3(256), 0, st, g);
  if (status != LLMK_OK) return status;
  const dim3 grid((unsigned)l.grid2);
  const bool many = s.splits > 2;
  return launch(l.steps == 1   ? (many ? k_lora_expand<1, true> : k_lora_expand<1, false>)
                : l.steps == 2 ? (many ? k_lora_expand<2, true> : k_lora_expand<2, false>)
                : l.steps == 4 ? k_lora_expand_high<4>
                               : k_lora_expand_high<8>,
                grid, dim3(256), 0, st, g);
}
