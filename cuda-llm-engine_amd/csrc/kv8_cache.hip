// Writing and reading the 8-bit KV cache (layout: kv8.hpp): the append of a pass's keys and values
// with the rotation of q and k on the way, and the read-back of cached rows as fp16.
//
// Append. The rotation of row at position pos, pair i < head_dim / 2 (element i with element i +
// head_dim / 2): angle = pos * inv_freq[i], c and s its cosine and sine, x1' = x1 c - x2 s, x2' =
// x2 c + x1 s. For k all of it is in 64 bits, so that its e4m3 codes, of which ties are close, are
// those of the definition (in 32 bits single ones are their neighbours: 28.6 and not 29.6 us for
// the prompts below, with read-back); for q c and s are rounded to 32 bits, the rest is done in
// them and rounded to fp16. k and v are rounded once, to e4m3 under the scale of their block. For
// the rows of the call that fall into one block (a page and kv head, K or V):
//   most  = the largest finite magnitude among them;
//   e     = the least exponent in [-15, 7] with most <= 448 * 2^e, or the block's own if that is
//           larger and the block holds tokens already (the first slot written is not its slot 0);
//   slots in front of the first one written are rounded again where e grew.
// So a block that is begun anew forgets its scale, and rows that are appended over others (drafted
// tokens that were refused) only ever find it as large as those needed.
//
// Work split: a window of 16 rows goes to a column of the grid, some blocks for its q, some for its
// K and V. The rows of the window that open a page, of their sequence or of the call, lead the rows
// that follow them in it. A wave holds all rows of a leader, in pieces of 16 values, and as many
// (kv head, K or V) side by side as fit its lanes: 16 rows of one at head_dim 64, 16 of single
// rows. So a window makes 16 to 32 such tasks whether it holds one prompt's rows or a decode
// step's, nothing is read twice, and the maximum is a few lane exchanges.
//
// What bounds it: for prompts HBM and what stands in front of a block's writes, its leaders, angles
// and maxima: 5 of up to 2001 rows take 25.5 us for 81 MB (22 where half of that is in the
// last-level cache), 12.5 at a large copy's 6.5 TB/s. Angles go by leader: where one leads 16 rows,
// 32 of the block's threads (64 at 128 dims) make all of them, and K and V are loaded behind that.
// For a decode step the way from the row starts over the lengths and tables to the scales, 4.7 us
// for one row and 6.0 for 256 of them (2.6 MB). A grid of one block for each row and head took 21.7
// us there, with read-back, and not 10.3.
#include <math.h>

#include "kv8.hpp"
#include "layer_ops.hpp"

namespace llmk {
namespace {

using namespace kv8;

// Cosine and sine of an angle, in 64 bits: the quarter turns are taken off in two parts (the angles
// of far positions lose their fraction in 32 bits), and what is left, at most pi / 4, goes through
// the series of both, which end below 2^-48 there. Their number, of up to 2^51, is the low bits of
// a sum with 1.5 * 2^52, whose last one is 1: a conversion to 32 bits would end at 2^31.
__device__ __forceinline__ double2 cos_sin(double angle) {
  constexpr double kWhole = 6755399441055744.0;
  const double turns = __builtin_fma(angle, 0.63661977236758134308, kWhole), k = turns - kWhole;
  double r = __builtin_fma(-k, 1.57079632679489655800, angle);
  r = __builtin_fma(-k, 6.12323399573676603587e-17, r);
  const double z = r * r;
  double s = -7.6471637318198164759e-13;  // (-1)^i / (2 i + 1)!, from i = 7 on down
  s = __builtin_fma(s, z, 1.6059043836821614599e-10);
  s = __builtin_fma(s, z, -2.5052108385441718775e-08);
  s = __builtin_fma(s, z, 2.7557319223985890653e-06);
  s = __builtin_fma(s, z, -1.9841269841269841270e-04);
  s = __builtin_fma(s, z, 8.3333333333333333333e-03);
  s = __builtin_fma(s, z, -1.6666666666666666667e-01);
  s = __builtin_fma(r * z, s, r);
  double c = -1.1470745597729724714e-11;  // (-1)^i / (2 i)!
  c = __builtin_fma(c, z, 2.0876756987868098979e-09);
  c = __builtin_fma(c, z, -2.7557319223985890653e-07);
  c = __builtin_fma(c, z, 2.4801587301587301587e-05);
  c = __builtin_fma(c, z, -1.3888888888888888889e-03);
  c = __builtin_fma(c, z, 4.1666666666666666667e-02);
  c = __builtin_fma(c, z, -0.5);
  c = __builtin_fma(c, z, 1.0);
  const int q = (int)(uint32_t)__builtin_bit_cast(uint64_t, turns) & 3;
  const double cq = (q & 1) ? s : c, sq = (q & 1) ? c : s;
  return make_double2(q == 1 || q == 2 ? -cq : cq, q >= 2 ? -sq : sq);
}

// x to 32 bits such that a later rounding to fewer than 23 is that of x itself, and so are
// comparisons with numbers of as few: the bits that do not fit are cut off, and where any was set
// the last one that does is set, too. They are the low 29 of the low half; infinities have none,
// and NaN stays NaN.
__device__ __forceinline__ float to_odd(double x) {
  const uint64_t b = __builtin_bit_cast(uint64_t, x);
  const uint32_t lo = (uint32_t)b;
  const uint32_t cut = (((lo & 0x1FFFFFFFu) + 0x1FFFFFFFu) | lo) & 0xE0000000u;
  return (float)__builtin_bit_cast(double, (b & 0xFFFFFFFF00000000ull) | cut);
}

struct AppendArgs {
  Batch batch;
  const f16* qkv;
  f16* q_out;
  uint8_t* pool[2];  // K, V
  float* scale[2];
  const float* inv_freq;
  int ld, n_heads, n_kv_heads;
};

constexpr int kWindow = 16, kQuarter = 4;  // rows of a column of the grid, and of a block for q

template <int HD>
__global__ void __launch_bounds__(256) k_kv8_append(const AppendArgs a, int kv_blocks) {
  constexpr int HALF = HD / 2, P = HD / 16;  // P pieces of a row: elements 8 p .. and HALF + 8 p ..
  constexpr int J = P * kPage / 64;          // rows of a lane where a page gets all 16
  __shared__ double2 turn[2 * kWindow][HALF];  // of the window's rows and what its last one leads
  __shared__ int seq_of[kWindow], lead[kWindow], slot_of[kWindow], tasks_before[kWindow + 1];
  __shared__ long long pos_of[kWindow];
  __shared__ size_t page_of[kWindow];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int window = blockIdx.x * kWindow, units = 2 * a.n_kv_heads;
  const int s0 = find_seq(a.batch.starts, a.batch.n_seqs, window);
  if (wave == 0) {
    const int row = window + lane;
    int s = -1, n = 0, slot = 0;  // n: rows that this one leads
    long long pos = -1;
    if (lane < kWindow && row < a.batch.n_rows && s0 >= 0)
      s = a.batch.starts ? find_seq_from(a.batch.starts, a.batch.n_seqs, s0, row)
                         : (row < a.batch.n_seqs ? row : -1);
    if (s >= 0) {
      const int r0 = a.batch.starts ? a.batch.starts[s] : row;
      const int r1 = a.batch.starts ? a.batch.starts[s + 1] : row + 1;
      pos = (long long)a.batch.lens[s] - (r1 - row);
      slot = (int)(pos & (kPage - 1));
      if (pos < 0 || pos >= (long long)a.batch.max_pages * kPage) {
        pos = -1;
      } else if (row == r0 || slot == 0) {
        n = kPage - slot;
        n = n < r1 - row ? n : r1 - row;
        n = n < a.batch.n_rows - row ? n : a.batch.n_rows - row;
        page_of[lane] = (size_t)a.batch.tables[(size_t)s * a.batch.max_pages + pos / kPage];
      }
    }
    int per = P;
    while (per < P * n && per < 64) per *= 2;
    int tasks = n > 0 ? (units + 64 / per - 1) / (64 / per) : 0;
    for (int d = 1; d < kWindow; d *= 2) {
      const int o = __shfl_up(tasks, d);
      if (lane >= d) tasks += o;
    }
    if (lane < kWindow) {
      seq_of[lane] = s;
      lead[lane] = n;
      slot_of[lane] = slot;
      pos_of[lane] = pos;
      tasks_before[lane + 1] = tasks;
      if (lane == 0) tasks_before[0] = 0;
    }
  }
  __syncthreads();

  if ((int)blockIdx.y >= kv_blocks) {  // q of 4 rows; zeros where a position lies outside the table
    const int r0 = ((int)blockIdx.y - kv_blocks) * kQuarter;
    for (int t = tid; t < kQuarter * HALF; t += 256)
      if (pos_of[r0 + t / HALF] >= 0)
        turn[t / HALF][t % HALF] =
            cos_sin((double)pos_of[r0 + t / HALF] * (double)a.inv_freq[t % HALF]);
    __syncthreads();
    const int per_row = a.n_heads * P;
    for (int t = tid; t < kQuarter * per_row; t += 256) {
      const int r = t / per_row, v = t % per_row, p = v % P;
      if (seq_of[r0 + r] < 0) continue;
      const bool in_table = pos_of[r0 + r] >= 0;
      const size_t row = (size_t)window + r0 + r, at = (size_t)(v / P) * HD + p * 8;
      const f16* src = a.qkv + row * a.ld + at;
      const f16x8 x1 = as_h8(ld16(src)), x2 = as_h8(ld16(src + HALF));
      f16x8 y1, y2;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const double2 cs = turn[r][p * 8 + e];
        const float u = (float)x1[e], w = (float)x2[e], c = (float)cs.x, s = (float)cs.y;
        y1[e] = in_table ? (f16)(u * c - w * s) : (f16)0;
        y2[e] = in_table ? (f16)(w * c + u * s) : (f16)0;
      }
      f16* dst = a.q_out + row * a.n_heads * HD + at;
      st16(dst, as_u4(y1));
      st16(dst + HALF, as_u4(y2));
    }
    return;
  }

  const int tasks = tasks_before[kWindow];
  if (tasks == 0) return;
  for (int t = tid; t < kWindow * HALF; t += 256) {  // leaders' rows, each by its leader
    const int g = t / HALF, i = t % HALF;
    for (int r = 0; r < lead[g]; ++r)
      turn[g + r][i] = cos_sin((double)(pos_of[g] + r) * (double)a.inv_freq[i]);
  }
  __syncthreads();
  for (int task = (int)blockIdx.y * 4 + wave; task < tasks; task += 4 * kv_blocks) {
    int g = 0;
    while (tasks_before[g + 1] <= task) ++g;
    const int n = lead[g], slot = slot_of[g];
    const size_t row = (size_t)window + g, page = page_of[g];
    int per = P;  // lanes of one unit, a (kv head, K or V): P for each row, rows to a power of two
    while (per < P * n && per < 64) per *= 2;
    const int mine = lane & (per - 1), r0 = mine / P, p = mine % P;
    const int unit = (task - tasks_before[g]) * (64 / per) + lane / per;
    const bool live = unit < units;
    const int side = live && unit >= a.n_kv_heads, h = live ? unit - side * a.n_kv_heads : 0;
    const f16* from =
        a.qkv + (size_t)(a.n_heads + side * a.n_kv_heads + h) * HD + 8 * p + row * a.ld;
    float* const scale = a.scale[side] + page * a.n_kv_heads + h;
    uint8_t* const block = a.pool[side] + (page * a.n_kv_heads + h) * (size_t)(kPage * HD);
    const int before = live && slot > 0 ? exponent_of(*scale) : kMinExp;
    float x[J][16];
    float most = 0.0f;
#pragma unroll
    for (int j = 0; j < J; ++j) {
      const int r = r0 + j * (64 / P);
      if (!live || r >= n) continue;
      const f16x8 x1 = as_h8(ld16(from + (size_t)r * a.ld));
      const f16x8 x2 = as_h8(ld16(from + (size_t)r * a.ld + HALF));
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float u = (float)x1[e], w = (float)x2[e];
        if (side == 0) {
          const double2 cs = turn[g + r][8 * p + e];
          x[j][e] = to_odd(__builtin_fma((double)u, cs.x, -((double)w * cs.y)));
          x[j][8 + e] = to_odd(__builtin_fma((double)w, cs.x, (double)u * cs.y));
        } else {
          x[j][e] = u;
          x[j][8 + e] = w;
        }
      }
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const float m = __builtin_fabsf(x[j][e]);
        most = m < INFINITY && m > most ? m : most;
      }
    }
    for (int d = 1; d < per; d *= 2) most = __builtin_fmaxf(most, __shfl_xor(most, d));
    int e = scale_exponent(most);
    e = e > before ? e : before;
    const float down = exp2_int(-e);
#pragma unroll
    for (int j = 0; j < J; ++j) {
      const int r = r0 + j * (64 / P);
      if (!live || r >= n) continue;
      uint8_t* dst = block + (slot + r) * HD + 8 * p;
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        uint2 v;
        v.x = to_e4m3(x[j][8 * k] * down, x[j][8 * k + 1] * down, x[j][8 * k + 2] * down,
                      x[j][8 * k + 3] * down);
        v.y = to_e4m3(x[j][8 * k + 4] * down, x[j][8 * k + 5] * down, x[j][8 * k + 6] * down,
                      x[j][8 * k + 7] * down);
        *reinterpret_cast<uint2*>(dst + k * HALF) = v;
      }
    }
    if (live && slot > 0 && e > before) {  // the tokens held already, under the new scale
      const float shift = exp2_int(before - e);
      for (int v = mine; v < slot * HD / 16; v += per) {
        u32x4 held = ld16(block + 16 * v);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const uint32_t b = elem(held, k);
          const f32x2 lo = __builtin_bit_cast(f32x2, __builtin_amdgcn_cvt_pk_f32_fp8(b, false));
          const f32x2 hi = __builtin_bit_cast(f32x2, __builtin_amdgcn_cvt_pk_f32_fp8(b, true));
          held[k] = to_e4m3(lo.x * shift, lo.y * shift, hi.x * shift, hi.y * shift);
        }
        st16(block + 16 * v, held);
      }
    }
    if (live && mine == 0) *scale = exp2_int(e);
  }
}

// Read-back: a block takes 16 rows of K or of V, a thread 8 values at a time, in the order of the
// output (a wave writes 1 KiB in a row; what it reads are 64-byte halves of lines whose other
// halves the neighbouring rows take), four of them in flight. Bound by HBM, two thirds of it
// writes: 64 sequences of up to 3001 rows, 314 MB, 59.7 us, 5.3 TB/s (48.5 where two such batches
// take turns and what is read stays in the last-level cache); in the order of the cache, which
// leaves lines half written, 82.4. 77 rows of one sequence 3.6 us, the way over starts, lengths,
// table and scale.
constexpr int kGatherRows = 16, kGatherFlight = 4;

struct GatherArgs {
  Batch batch;
  const uint8_t* pool[2];
  const float* scale[2];
  f16* out[2];
  int n_kv_heads;
  FastDiv per_row;  // 8-value pieces of a row
};

template <int HD>
__global__ void __launch_bounds__(256) k_kv8_gather(const GatherArgs a) {
  constexpr int P = HD / 8;
  __shared__ long long block_of[kGatherRows];  // page, -1: no position, -2: a row of no sequence
  __shared__ int slot_of[kGatherRows];
  const int row0 = blockIdx.x * kGatherRows, tid = threadIdx.x;
  const int s0 = find_seq(a.batch.starts, a.batch.n_seqs, row0);
  if (tid < kGatherRows) {
    const int row = row0 + tid;
    int s = -1;
    if (row < a.batch.n_rows && s0 >= 0)
      s = a.batch.starts ? find_seq_from(a.batch.starts, a.batch.n_seqs, s0, row)
                         : (row < a.batch.n_seqs ? row : -1);
    long long page = -2;
    if (s >= 0) {
      const long long back = a.batch.starts ? (long long)a.batch.starts[s + 1] - row : 1;
      const long long pos = a.batch.lens[s] - back;
      const bool in_table = pos >= 0 && pos < (long long)a.batch.max_pages * kPage;
      page = in_table ? a.batch.tables[(size_t)s * a.batch.max_pages + pos / kPage] : -1;
      slot_of[tid] = (int)(pos & (kPage - 1));
    }
    block_of[tid] = page;
  }
  __syncthreads();
  const int side = blockIdx.y, n = kGatherRows * (int)a.per_row.d;
  for (int t0 = tid; t0 < n; t0 += 256 * kGatherFlight) {
    uint2 bytes[kGatherFlight];
    float scale[kGatherFlight];
    int row[kGatherFlight];
#pragma unroll
    for (int k = 0; k < kGatherFlight; ++k) {
      const int t = t0 + 256 * k;
      const int r = t < n ? (int)fdiv((uint32_t)t, a.per_row) : 0;
      const int v = t < n ? t - r * (int)a.per_row.d : 0;
      const long long page = t < n ? block_of[r] : -2;
      row[k] = page == -2 ? -1 : r;
      bytes[k] = make_uint2(0, 0);
      scale[k] = 1.0f;
      if (page >= 0) {
        const size_t block = (size_t)page * a.n_kv_heads + v / P;
        bytes[k] = *reinterpret_cast<const uint2*>(
            a.pool[side] + (block * kPage + slot_of[r]) * HD + 8 * (v % P));
        scale[k] = a.scale[side][block];
      }
    }
#pragma unroll
    for (int k = 0; k < kGatherFlight; ++k) {
      if (row[k] < 0) continue;
      const int v = t0 + 256 * k - row[k] * (int)a.per_row.d;
      u32x4 y;
      y[0] = __builtin_bit_cast(uint32_t, from_e4m3<false>(bytes[k].x, scale[k]));
      y[1] = __builtin_bit_cast(uint32_t, from_e4m3<true>(bytes[k].x, scale[k]));
      y[2] = __builtin_bit_cast(uint32_t, from_e4m3<false>(bytes[k].y, scale[k]));
      y[3] = __builtin_bit_cast(uint32_t, from_e4m3<true>(bytes[k].y, scale[k]));
      st16_stream(a.out[side] + ((size_t)(row0 + row[k]) * a.per_row.d + v) * 8, y);
    }
  }
}

int check_batch(int n_rows, int n_seqs, int max_pages, int page_size, int n_kv_heads, int head_dim,
                const int32_t* row_starts) {
  if (n_rows < 0 || n_seqs < 0 || max_pages <= 0 || n_kv_heads <= 0 || head_dim <= 0)
    return LLMK_ERR_INVALID_VALUE;
  if (!row_starts && n_rows != n_seqs) return LLMK_ERR_INVALID_VALUE;
  if (page_size != kPage || (head_dim != 64 && head_dim != 128)) return LLMK_ERR_SHAPE;
  return LLMK_OK;
}

}  // namespace
}  // namespace llmk

using namespace llmk;

extern "C" int llmk_kv8_append(const uint16_t* qkv, int ld, uint16_t* q_out, uint8_t* k_pool,
                               float* k_scale, uint8_t* v_pool, float* v_scale,
                               const int32_t* block_tables, const int32_t* row_starts,
                               const int32_t* seq_lens, const float* inv_freq, int n_rows,
                               int n_seqs, int max_pages, int page_size, int n_heads,
                               int n_kv_heads, int head_dim, void* stream) {
  const int st =
      check_batch(n_rows, n_seqs, max_pages, page_size, n_kv_heads, head_dim, row_starts);
  if (st != LLMK_OK) return st;
  if (n_heads <= 0) return LLMK_ERR_INVALID_VALUE;
  if ((long long)ld < ((long long)n_heads + 2LL * n_kv_heads) * head_dim || ld % 8 != 0)
    return LLMK_ERR_SHAPE;
  if (n_rows == 0 || n_seqs == 0) return LLMK_OK;
  const size_t windows = ceil_div((size_t)n_rows, (size_t)kWindow);
  if (!grid_takes(windows, 256)) return LLMK_ERR_UNSUPPORTED;
  if (!qkv || !q_out || !k_pool || !k_scale || !v_pool || !v_scale || !block_tables || !seq_lens ||
      !inv_freq)
    return LLMK_ERR_INVALID_VALUE;
  if (!aligned16(qkv) || !aligned16(q_out) || !aligned16(k_pool) || !aligned16(v_pool))
    return LLMK_ERR_ALIGNMENT;
  AppendArgs a;
  a.batch = kv8::Batch{block_tables, row_starts, seq_lens, n_rows, n_seqs, max_pages};
  a.qkv = reinterpret_cast<const f16*>(qkv);
  a.q_out = reinterpret_cast<f16*>(q_out);
  a.pool[0] = k_pool;
  a.pool[1] = v_pool;
  a.scale[0] = k_scale;
  a.scale[1] = v_scale;
  a.inv_freq = inv_freq;
  a.ld = ld;
  a.n_heads = n_heads;
  a.n_kv_heads = n_kv_heads;
  // a block for K and V takes four tasks at a time of the window's 16 to 32 at 8 kv heads
  const int kv_blocks = (n_kv_heads + 1) / 2 < 32 ? (n_kv_heads + 1) / 2 : 32;
  const dim3 grid((unsigned)windows, kv_blocks + kWindow / kQuarter);
  return launch(head_dim == 64 ? k_kv8_append<64> : k_kv8_append<128>, grid, dim3(256), 0,
                static_cast<hipStream_t>(stream), a, kv_blocks);
}

extern "C" int llmk_kv8_gather(const uint8_t* k_pool, const float* k_scale, const uint8_t* v_pool,
                               const float* v_scale, const int32_t* block_tables,
                               const int32_t* row_starts, const int32_t* seq_lens,
                               uint16_t* k_out, uint16_t* v_out, int n_rows, int n_seqs,
                               int max_pages, int page_size, int n_kv_heads, int head_dim,
                               void* stream) {
  const int st =
      check_batch(n_rows, n_seqs, max_pages, page_size, n_kv_heads, head_dim, row_starts);
  if (st != LLMK_OK) return st;
  if (n_kv_heads > 65536) return LLMK_ERR_UNSUPPORTED;  // a block's share is counted in 32 bits
  if (n_rows == 0 || n_seqs == 0) return LLMK_OK;
  const size_t blocks = ceil_div((size_t)n_rows, (size_t)kGatherRows);
  if (!grid_takes(blocks, 256)) return LLMK_ERR_UNSUPPORTED;
  if (!k_pool || !k_scale || !v_pool || !v_scale || !block_tables || !seq_lens || !k_out || !v_out)
    return LLMK_ERR_INVALID_VALUE;
  if (!aligned16(k_pool) || !aligned16(v_pool) || !aligned16(k_out) || !aligned16(v_out))
    return LLMK_ERR_ALIGNMENT;
  GatherArgs a;
  a.batch = kv8::Batch{block_tables, row_starts, seq_lens, n_rows, n_seqs, max_pages};
  a.pool[0] = k_pool;
  a.pool[1] = v_pool;
  a.scale[0] = k_scale;
  a.scale[1] = v_scale;
  a.out[0] = reinterpret_cast<f16*>(k_out);
  a.out[1] = reinterpret_cast<f16*>(v_out);
  a.n_kv_heads = n_kv_heads;
  a.per_row = make_fastdiv((uint32_t)n_kv_heads * (uint32_t)head_dim / 8);
  return launch(head_dim == 64 ? k_kv8_gather<64> : k_kv8_gather<128>,
                dim3((unsigned)blocks, 2), dim3(256), 0, static_cast<hipStream_t>(stream), a);
}
