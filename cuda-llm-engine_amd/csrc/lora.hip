// Low-rank adapters of a batch's sequences beside a shared projection:
//   y[r, :] += scale_a B_a h, h = A_a x[r, :], a the adapter of row r's sequence.
//
// Two launches of matrix products, tiles of 16 rows that have the same adapter, so that its weights are
// read once for them: k_lora_shrink finds the tiles and computes h, k_lora_expand adds B_a h to y.
//
// Tiles. Sequences are taken 256 at a time (a window); those of a window with the same adapter are a
// group, in the order of their first ones, and a group's rows, in order, are cut into tiles of 16. Every
// block of k_lora_shrink finds its tile by itself: adapters into a hash table in LDS, whose slots collect
// the members as bits; counts of tiles summed up by the group's first member. That takes about a
// microsecond beside the loads of ids and starts, which a launch of its own would have to wait for too.
// What a block finds does not depend on the order in which threads reach the table. Window w's tiles
// begin at slot starts[256 w] / 16 + w * (groups + 1), which leaves room for all of them: slots without a
// tile are noted as such.
//
// Between the products h is held in fp32 (the blocks of a tile that share out in_features leave a sum
// each) and given to the matrix instructions as two fp16: h * 2^-e, with 2^e such that the row's largest
// is from 2^14 to 2^15, rounded, and what that lost. That keeps 22 bits relative to the row's largest, and the sum
// is multiplied by scale * 2^e in fp32. So neither large nor small values of h leave fp16's range.
#include "kv8.hpp"

namespace llmk {
namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));

constexpr int kParts = 8, kMaxRank = 256;
constexpr int kWindow = 256, kHash = 512;
constexpr int kRows = 16;   // of a tile
constexpr int kNote = 32;   // ints of a tile's note: adapter (-1: no tile), then its rows (-1: none)
constexpr int kChunk = 256;  // of in_features that a wave takes at a time
constexpr int kGroups = 4;  // of 16 ranks that it accumulates at a time

struct LoraArgs {
  const f16 *x, *a, *b;
  const int *ranks, *ids, *starts;
  const float* scales;
  f16* y;
  int* notes;   // workspace: [slots, kNote]
  float* h;     // [splits, slots, kRows, n_parts * max_rank]
  int part_end[kParts], chunk_end[kParts];  // columns, and blocks of k_lora_expand, up to each part's end
  int ldx, ldy, n_parts, n_rows, n_seqs, n_adapters, max_rank, in;
  int slots, splits, groups, windows, per_block;
};

__device__ __forceinline__ int first_row(const LoraArgs& g, int s) {
  const int r = g.starts ? g.starts[s] : s;
  return r < 0 ? 0 : r < g.n_rows ? r : g.n_rows;
}

__device__ __forceinline__ int slot_of_window(const LoraArgs& g, int w) {
  return first_row(g, min(w * kWindow, g.n_seqs)) / kRows + w * (g.groups + 1);
}

__device__ __forceinline__ int rank_of(const LoraArgs& g, int a) {
  return g.ranks ? min(g.ranks[a], g.max_rank) : g.max_rank;
}

__device__ __forceinline__ int wave_scan(int v) {  // inclusive
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int d = 1; d < 64; d *= 2) {
    const int o = __shfl_up(v, d);
    if (lane >= d) v += o;
  }
  return v;
}

// The sum of v over the threads in front, of 256. part: four ints that no thread still reads.
__device__ __forceinline__ int block_scan(int v, int* part) {
  const int wave = threadIdx.x >> 6, in = wave_scan(v);
  if ((threadIdx.x & 63) == 63) part[wave] = in;
  __syncthreads();
  int before = 0;
#pragma unroll
  for (int w = 0; w < 3; ++w) before += w < wave ? part[w] : 0;
  return before + in - v;
}

struct Plan {
  int key[kHash];            // the adapter of a slot of the table, -1: none
  int rows[kHash];           // its rows
  int first[kHash];          // its first member
  int part[2][4];
  int adapter, group, from;  // of the tile: its group's table slot, and its first row among the group's
  int row[kRows];
};

// Finds tile `slot` with 256 threads: its adapter (-1: there is none) and rows, in p.
__device__ __forceinline__ void find_tile(const LoraArgs& g, int slot, Plan& p) {
  const int tid = threadIdx.x;
  int w = 0;
  for (int hi = g.windows; hi - w > 1;) {  // the last window that begins at or before the slot
    const int mid = (w + hi) / 2;
    if (slot_of_window(g, mid) <= slot) w = mid; else hi = mid;
  }
  const int s = w * kWindow + tid;
  int id = -1, r0 = 0, rows = 0;
  if (s < g.n_seqs) {
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
  __syncthreads();
  int at = -1;
  if (id >= 0) {  // at most kWindow adapters in kHash slots: the search ends
    at = (int)(((unsigned)id * 2654435761u) >> 23);
    for (;;) {
      const int was = atomicCAS(&p.key[at], -1, id);
      if (was == -1 || was == id) break;
      at = (at + 1) & (kHash - 1);
    }
    atomicAdd(&p.rows[at], rows);
    atomicMin(&p.first[at], tid);
  }
  __syncthreads();
  const bool leads = at >= 0 && p.first[at] == tid;
  const int tiles = leads ? (p.rows[at] + kRows - 1) / kRows : 0;
  const int begin = block_scan(tiles, p.part[0]);
  if (leads && tile >= begin && tile < begin + tiles) {
    p.adapter = id;
    p.group = at;
    p.from = (tile - begin) * kRows;
  }
  __syncthreads();
  if (p.adapter < 0) return;
  const bool mine = at == p.group;
  const int before = block_scan(mine ? rows : 0, p.part[1]) - p.from;
  if (mine)
    for (int i = max(-before, 0); i < rows && before + i < kRows; ++i) p.row[before + i] = r0 + i;
  __syncthreads();
}

// h of a tile: D[rank, row] = A[rank, k] x[row, k], by waves that take 256 of in_features at a time.
__global__ void __launch_bounds__(256) k_lora_shrink(const LoraArgs g) {
  __shared__ Plan p;
  __shared__ f32x4 sum[3][kGroups][64];
  const int slot = blockIdx.x, split = blockIdx.y;
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, n = lane & 15, q = lane >> 4;
  find_tile(g, slot, p);
  const int a = p.adapter;
  if (split == 0) {
    if (threadIdx.x == 0) g.notes[(size_t)slot * kNote] = a;
    if (threadIdx.x < kRows) g.notes[(size_t)slot * kNote + 1 + threadIdx.x] = p.row[threadIdx.x];
  }
  if (a < 0) return;
  const int rank = rank_of(g, a);
  if (rank <= 0) return;
  const int per_part = (rank + 15) / 16, all = g.n_parts * per_part;
  const int row = p.row[n] >= 0 ? p.row[n] : p.row[0];  // a row that is none gives what nobody reads
  const f16* x = g.x + (size_t)row * g.ldx + 8 * q;
  const size_t width = (size_t)g.n_parts * g.max_rank;
  float* out = g.h + ((size_t)split * g.slots + slot) * kRows * width + n * width + 4 * q;
  for (int g0 = 0; g0 < all; g0 += kGroups) {
    f32x4 acc[kGroups];
    const f16* w[kGroups];
#pragma unroll
    for (int i = 0; i < kGroups; ++i) {
      acc[i] = f32x4{0.f, 0.f, 0.f, 0.f};
      const int gi = min(g0 + i, all - 1), part = gi / per_part;
      const int j = min((gi - part * per_part) * 16 + n, rank - 1);
      w[i] = g.a + (((size_t)a * g.n_parts + part) * g.max_rank + j) * g.in + 8 * q;
    }
    for (int c = split * 4 + wave; c * kChunk < g.in; c += 4 * g.splits) {
      const int k0 = c * kChunk;
      u32x4 xf[8];
#pragma unroll
      for (int t = 0; t < 8; ++t) {
        const int k = k0 + 32 * t;
        xf[t] = k + 8 * q < g.in ? ld16(x + k) : u32x4{0, 0, 0, 0};
      }
#pragma unroll
      for (int i = 0; i < kGroups; ++i) {
        if (g0 + i >= all) break;
        u32x4 wf[8];
#pragma unroll
        for (int t = 0; t < 8; ++t) {
          const int k = k0 + 32 * t;
          wf[t] = k + 8 * q < g.in ? ld16(w[i] + k) : u32x4{0, 0, 0, 0};
        }
#pragma unroll
        for (int t = 0; t < 8; ++t)
          acc[i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(as_h8(wf[t]), as_h8(xf[t]), acc[i], 0, 0, 0);
      }
    }
    // the four waves' sums, the first one's last
    if (g0) __syncthreads();
    if (wave > 0)
#pragma unroll
      for (int i = 0; i < kGroups; ++i) sum[wave - 1][i][lane] = acc[i];
    __syncthreads();
    if (wave == 0)
#pragma unroll
      for (int i = 0; i < kGroups; ++i) {
        if (g0 + i >= all) break;
        acc[i] = (acc[i] + sum[0][i][lane]) + (sum[1][i][lane] + sum[2][i][lane]);
        const int part = (g0 + i) / per_part, j = (g0 + i - part * per_part) * 16;
        if (j + 4 * q < g.max_rank)
          *reinterpret_cast<f32x4*>(out + (size_t)part * g.max_rank + j) = acc[i];
      }
  }
}

// y of a tile's rows and a block's columns: D[column, row] = B[column, j] h[row, j], in steps of 32 ranks (KS
// at most). The columns of a wave are taken 32 at a time by two products, whose rows of B are chosen such
// that a lane gets eight columns side by side.
template <int KS>
__global__ void __launch_bounds__(256) k_lora_expand(const LoraArgs g) {
  constexpr int TILES = KS <= 2 ? 8 : 16 / KS, PAIRS = TILES / 2;  // products of a wave
  constexpr int LD = 32 * KS + 8;                                  // of a row in LDS
  __shared__ __attribute__((aligned(16))) f16 hi[kRows * LD], lo[kRows * LD];
  __shared__ float power[kRows];
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, n = lane & 15, q = lane >> 4;
  int part = 0;
  while ((int)blockIdx.y >= g.chunk_end[part]) ++part;
  const int chunk = blockIdx.y - (part ? g.chunk_end[part - 1] : 0);
  const int end = g.part_end[part], out = g.part_end[g.n_parts - 1];
  const int c0 = (part ? g.part_end[part - 1] : 0) + (chunk * 4 + wave) * 16 * TILES;
  const size_t width = (size_t)g.n_parts * g.max_rank;
  u32x4 bf[TILES][KS];
  int loaded = -1, rank = 0;
  float scale = 0.f;
  for (int i = 0; i < g.per_block; ++i) {
    const int slot = blockIdx.x * g.per_block + i;
    if (slot >= g.slots) break;
    const int* note = g.notes + (size_t)slot * kNote;
    const int a = note[0], row = note[1 + n];
    if ((unsigned)a >= (unsigned)g.n_adapters) continue;
    if (a != loaded) {
      loaded = a;
      rank = rank_of(g, a);
      scale = g.scales ? g.scales[a] : 1.f;
      if (rank > 0)
#pragma unroll
        for (int t = 0; t < TILES; ++t) {
          const int c = min(c0 + 32 * (t / 2) + 8 * (n / 4) + 4 * (t & 1) + n % 4, end - 1);
          const f16* b = g.b + ((size_t)a * out + c) * g.max_rank + 8 * q;
#pragma unroll
          for (int s = 0; s < KS; ++s) {
            const int k = 32 * s + 8 * q;
            f16x8 v = (f16x8)(f16)0;
            if (k < rank) v = as_h8(ld16(b + 32 * s));
            if (k + 8 > rank)
#pragma unroll
              for (int e = 0; e < 8; ++e) v[e] = k + e < rank ? v[e] : (f16)0;
            bf[t][s] = as_u4(v);
          }
        }
    }
    if (rank <= 0) continue;
    f16* y = g.y + (size_t)((unsigned)row < (unsigned)g.n_rows ? row : 0) * g.ldy + c0 + 8 * q;
    u32x4 old[PAIRS];
#pragma unroll
    for (int t = 0; t < PAIRS; ++t)
      if ((unsigned)row < (unsigned)g.n_rows && c0 + 32 * t + 8 * q < end) old[t] = ld16(y + 32 * t);
    // h into LDS: 16 threads a row, eight ranks each
    lds_barrier();
    {
      const int r = threadIdx.x >> 4, piece = threadIdx.x & 15;
      constexpr int PIECES = (KS * 4 + 15) / 16;
      float v[PIECES][8], most = 0.f;
      const float* h = g.h + ((size_t)slot * kRows + r) * width + (size_t)part * g.max_rank;
#pragma unroll
      for (int m = 0; m < PIECES; ++m) {
        const int k = 8 * (piece + 16 * m);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[m][e] = 0.f;
        if (k < rank)
          for (int s = 0; s < g.splits; ++s) {
            const f32x4* from =
                reinterpret_cast<const f32x4*>(h + (size_t)s * g.slots * kRows * width + k);
            const f32x4 u = from[0], w = from[1];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              v[m][e] += u[e];
              v[m][e + 4] += w[e];
            }
          }
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          v[m][e] = k + e < rank ? v[m][e] : 0.f;
          const float mag = __builtin_fabsf(v[m][e]);
          most = mag < INFINITY ? __builtin_fmaxf(most, mag) : most;
        }
      }
#pragma unroll
      for (int d = 1; d < 16; d *= 2) most = __builtin_fmaxf(most, __shfl_xor(most, d));
      // 2^e: the largest becomes 2^14 or more, below 2^15
      int e = (int)(__builtin_bit_cast(uint32_t, most) >> 23) - 127 - 14;
      e = e < -100 ? -100 : e;
      const float down = kv8::exp2_int(-e);
      if (piece == 0) power[r] = kv8::exp2_int(e);
#pragma unroll
      for (int m = 0; m < PIECES; ++m) {
        const int k = 8 * (piece + 16 * m);
        f16x8 big, rest;
#pragma unroll
        for (int i2 = 0; i2 < 8; ++i2) {
          const float u = v[m][i2] * down;
          big[i2] = (f16)u;
          rest[i2] = __builtin_fabsf(u) < INFINITY ? (f16)(u - (float)big[i2]) : (f16)0;
        }
        if (k < 32 * KS) {
          *reinterpret_cast<f16x8*>(hi + r * LD + k) = big;
          *reinterpret_cast<f16x8*>(lo + r * LD + k) = rest;
        }
      }
    }
    lds_barrier();
    f16x8 hf[KS], lf[KS];
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      hf[s] = *reinterpret_cast<const f16x8*>(hi + n * LD + 32 * s + 8 * q);
      lf[s] = *reinterpret_cast<const f16x8*>(lo + n * LD + 32 * s + 8 * q);
    }
    const float by = scale * power[n];
#pragma unroll
    for (int t = 0; t < PAIRS; ++t) {
      f32x4 d[2];
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        d[j] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int s = 0; s < KS; ++s) {
          d[j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(as_h8(bf[2 * t + j][s]), hf[s], d[j], 0, 0, 0);
          d[j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(as_h8(bf[2 * t + j][s]), lf[s], d[j], 0, 0, 0);
        }
      }
      if ((unsigned)row < (unsigned)g.n_rows && c0 + 32 * t + 8 * q < end) {
        f16x8 v = as_h8(old[t]);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = (f16)((float)v[e] + by * d[e / 4][e % 4]);
        st16(y + 32 * t, as_u4(v));
      }
    }
  }
}

// What a call takes of the chip and the workspace, by its sizes alone.
struct Shape {
  int groups, windows, slots, splits;
};
Shape shape_of(int n_rows, int n_seqs, int n_adapters, int in) {
  Shape s;
  s.groups = n_seqs < kWindow ? n_seqs : kWindow;
  if (n_adapters < s.groups) s.groups = n_adapters;
  s.windows = (n_seqs + kWindow - 1) / kWindow;
  s.slots = n_rows / kRows + s.windows * (s.groups + 1);
  const int most = (in + 4 * kChunk - 1) / (4 * kChunk);
  s.splits = (512 + s.slots - 1) / s.slots;
  if (s.splits > most) s.splits = most;
  return s;
}

}  // namespace
}  // namespace llmk

using namespace llmk;

extern "C" size_t llmk_lora_add_workspace_floats(int n_rows, int n_seqs, int n_adapters, int max_rank,
                                                 int in_features, int n_parts) {
  if (n_rows <= 0 || n_seqs <= 0 || n_adapters <= 0 || max_rank <= 0 || in_features <= 0 ||
      n_parts <= 0)
    return 0;
  const Shape s = shape_of(n_rows, n_seqs, n_adapters, in_features);
  return (size_t)s.slots * (kNote + (size_t)s.splits * kRows * n_parts * max_rank);
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
  const int steps = (max_rank + 31) / 32, ks = steps <= 2 ? steps : steps <= 4 ? 4 : 8;
  const int columns = ks <= 2 ? 512 : 1024 / ks;  // of a block
  LoraArgs g{};
  for (int p = 0; p < n_parts; ++p) {
    const int begin = p ? part_ends[p - 1] : 0;
    if (part_ends[p] <= begin) return LLMK_ERR_INVALID_VALUE;
    if (part_ends[p] % 8) return LLMK_ERR_SHAPE;
    g.part_end[p] = part_ends[p];
    g.chunk_end[p] = (p ? g.chunk_end[p - 1] : 0) + (int)ceil_div(part_ends[p] - begin, columns);
  }
  if (in_features % 8 || max_rank % 8 || ldx % 8 || ldy % 8 || ldx < in_features ||
      ldy < part_ends[n_parts - 1])
    return LLMK_ERR_SHAPE;
  if (max_rank > kMaxRank || n_rows > (1 << 20) || n_seqs > (1 << 20) || in_features > (1 << 24) ||
      g.chunk_end[n_parts - 1] > 65535)
    return LLMK_ERR_UNSUPPORTED;
  if (n_rows == 0 || n_seqs == 0 || n_adapters == 0) return LLMK_OK;
  if (!x || !a || !b || !adapter_ids || !y || !workspace) return LLMK_ERR_INVALID_VALUE;
  if (!aligned16(x) || !aligned16(a) || !aligned16(b) || !aligned16(y) || !aligned16(workspace))
    return LLMK_ERR_ALIGNMENT;
  const Shape s = shape_of(n_rows, n_seqs, n_adapters, in_features);
  g.x = reinterpret_cast<const f16*>(x);
  g.a = reinterpret_cast<const f16*>(a);
  g.b = reinterpret_cast<const f16*>(b);
  g.ranks = ranks;
  g.ids = adapter_ids;
  g.starts = row_starts;
  g.scales = scales;
  g.y = reinterpret_cast<f16*>(y);
  g.notes = reinterpret_cast<int*>(workspace);
  g.h = workspace + (size_t)s.slots * kNote;
  g.ldx = ldx;
  g.ldy = ldy;
  g.n_parts = n_parts;
  g.n_rows = n_rows;
  g.n_seqs = n_seqs;
  g.n_adapters = n_adapters;
  g.max_rank = max_rank;
  g.in = in_features;
  g.slots = s.slots;
  g.splits = s.splits;
  g.groups = s.groups;
  g.windows = s.windows;
  hipStream_t st = static_cast<hipStream_t>(stream);
  const int status = launch(k_lora_shrink, dim3(s.slots, s.splits), dim3(256), 0, st, g);
  if (status != LLMK_OK) return status;
  const int chunks = g.chunk_end[n_parts - 1];
  g.per_block = 1;
  while (g.per_block < 8 && (long long)s.slots * chunks / (2 * g.per_block) >= 2048) g.per_block *= 2;
  const dim3 grid(ceil_div(s.slots, g.per_block), chunks);
  return launch(ks == 1 ? k_lora_expand<1> : ks == 2 ? k_lora_expand<2>
                : ks == 4 ? k_lora_expand<4> : k_lora_expand<8>,
                grid, dim3(256), 0, st, g);
}
