// Rotary positions of either layout, of part of a head, with a frequency table and a scale for each
// row; where the rows lie, or on their way into the paged cache.
//
// x1' = s (x1 cos t - x2 sin t), x2' = s (x2 cos t + x1 sin t) for the elements that turn together, t =
// position * inv_freq in 64 bits: an angle of a far position has lost its fraction in 32. The cosine and
// sine, times s, are rounded to fp32 once for all heads of the row, the products and their sum are fp32
// and the result is rounded to fp16: off by 2^-11 of itself and 2^-22 of |x1| + |x2|.
//
// A head's rotated part is cut into units of 16 elements, two 16-byte vectors that a thread turns by
// itself, without its neighbours: vectors u and u + rotary_dim / 16. As halves they are each other's
// partners; as pairs each holds four pairs. Either way a wave's loads cover whole lines.
//
// Bound by bytes, each once each way; a 64-bit cosine and sine take some 60 instructions a pair of a row, which is why
// they are computed once a row for all its heads and while the data is on its way. Measured (one MI355X, inputs from
// HBM, the floor at 6 TB/s), us: 1 row 2.1 (one launch); 4001 rows of 40 heads of 64 in place 10.2 (6.8: 41 MB at 4
// TB/s; not the memory's bound, as more units a thread take 9.5); 256 rows into the cache 3.6 (0.5); 2001 rows of 28 +
// 2 x 4 heads of 128 into the cache 10.2 (6.2: 37 MB, of which a plain copy takes 7). What is no whole vectors is turned
// pair by pair: 4001 rows of 40 heads of 64 with 24 elements turned take 11.9 (2.6), with all of them at odd addresses
// 22.3 (6.8), one row 2.5.
#include "angles.hpp"
#include "layer_ops.hpp"
#include "overlap.hpp"

namespace llmk {
namespace {

struct RotaryArgs {
  const f16 *q, *k, *v;  // row r at r * ld of each
  f16 *q_out, *k_out, *v_out;
  const int *positions, *table_ids, *tables;
  const float *inv_freq, *scales;
  int ldq, ldk, ldq_out, ldk_out;  // ldk_out: of a row of the pool (in place: ldk)
  int n_rows, n_heads, n_kv_heads, head_dim, rotary_dim, n_tables;
  int max_pages, page_size;
  int rows, chunks, per_row;  // of a block; blocks of a row (where it is wide), units of a row
  FastDiv by_row, by_unit, by_half;
};

// What the turn of pair i of a row is made of, and the turn: (scale cos, scale sin).
struct Angle {
  int pos;
  float freq, scale;
};
__device__ __forceinline__ Angle angle_of(const RotaryArgs& a, int row, int i) {
  Angle x;
  x.pos = a.positions[row];
  int t = a.table_ids ? a.table_ids[row] : 0;
  t = (unsigned)t < (unsigned)a.n_tables ? t : 0;
  x.freq = a.inv_freq[(size_t)t * (a.rotary_dim / 2) + i];
  x.scale = a.scales ? a.scales[t] : 1.f;
  return x;
}
__device__ __forceinline__ float2 turn_of(Angle x) {
  const double2 cs = cos_sin((double)x.pos * (double)x.freq);
  return make_float2((float)(cs.x * (double)x.scale), (float)(cs.y * (double)x.scale));
}

// The pool row (page * page_size + token) of a row, -1 where it has none.
__device__ __forceinline__ long long pool_row_of(const RotaryArgs& a, int row) {
  const int pos = a.positions[row];
  if (pos < 0 || pos / a.page_size >= a.max_pages) return -1;
  const int page = a.tables[(size_t)row * a.max_pages + pos / a.page_size];
  return page < 0 ? -1 : (long long)page * a.page_size + pos % a.page_size;
}

template <bool PAIRS>
__device__ __forceinline__ void turn(f16x8& x, f16x8& y, const float2* lo, const float2* hi) {
  if (PAIRS) {  // lo, hi: the four turns of x's pairs and of y's
#pragma unroll
    for (int e = 0; e < 8; e += 2) {
      const float2 c = lo[e / 2], d = hi[e / 2];
      const float x1 = (float)x[e], x2 = (float)x[e + 1], y1 = (float)y[e], y2 = (float)y[e + 1];
      x[e] = (f16)(x1 * c.x - x2 * c.y);
      x[e + 1] = (f16)(x2 * c.x + x1 * c.y);
      y[e] = (f16)(y1 * d.x - y2 * d.y);
      y[e + 1] = (f16)(y2 * d.x + y1 * d.y);
    }
  } else {  // lo: the eight turns of x's elements with y's
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float2 c = lo[e];
      const float x1 = (float)x[e], x2 = (float)y[e];
      x[e] = (f16)(x1 * c.x - x2 * c.y);
      y[e] = (f16)(x2 * c.x + x1 * c.y);
    }
  }
}

// U units a thread. What the turns are made of is loaded first, then the data: the turns are computed while that
// is on its way, and it is turned and stored behind the barrier.
template <bool PAIRS, bool SCATTER, int U>
__global__ void __launch_bounds__(512) k_rotary(const RotaryArgs a) {
  extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
  float2* turns = reinterpret_cast<float2*>(smem);  // [row][pair]
  const int tid = threadIdx.x, threads = blockDim.x, half = a.rotary_dim / 2, R = a.rotary_dim / 16;
  const int group = blockIdx.x / a.chunks, row0 = group * a.rows, rows = min(a.rows, a.n_rows - row0);
  const int unit0 = (blockIdx.x - group * a.chunks) * threads * U + tid;
  long long* pool_row = reinterpret_cast<long long*>(turns + (size_t)a.rows * half);
  const int n_turns = rows * half;
  Angle angle;
  if (tid < n_turns) {
    const int r = (int)fdiv(tid, a.by_half);
    angle = angle_of(a, row0 + r, tid - r * half);
  }
  if (SCATTER && tid < rows) pool_row[tid] = pool_row_of(a, row0 + tid);
  // a head's units: R that turn and, where rows move, those behind them; v's heads move whole
  int r[U], head[U], i[U], j[U];
  bool moves[U];
  f16x8 x[U], y[U];
#pragma unroll
  for (int m = 0; m < U; ++m) {
    const int unit = unit0 + m * threads;
    r[m] = (int)fdiv(unit, a.by_row);
    const int rest = unit - r[m] * a.per_row;
    head[m] = (int)fdiv(rest, a.by_unit);
    const int u = rest - head[m] * (int)a.by_unit.d, kv = head[m] - a.n_heads, vv = kv - a.n_kv_heads;
    moves[m] = SCATTER && (u >= R || vv >= 0);
    i[m] = moves[m] ? 2 * u : u;
    j[m] = moves[m] ? 2 * u + 1 : u + R;
    if (r[m] < rows) {
      const size_t row = row0 + r[m];
      const f16* src = kv < 0               ? a.q + row * a.ldq + (size_t)head[m] * a.head_dim
                       : SCATTER && vv >= 0 ? a.v + row * a.ldk + (size_t)vv * a.head_dim
                                            : a.k + row * a.ldk + (size_t)kv * a.head_dim;
      x[m] = as_h8(ld16_stream(src + 8 * i[m]));
      y[m] = as_h8(ld16_stream(src + 8 * j[m]));
    }
  }
  if (tid < n_turns) turns[tid] = turn_of(angle);
  for (int e = tid + threads; e < n_turns; e += threads) {
    const int q = (int)fdiv(e, a.by_half);
    turns[e] = turn_of(angle_of(a, row0 + q, e - q * half));
  }
  lds_barrier();
#pragma unroll
  for (int m = 0; m < U; ++m) {
    if (r[m] >= rows) return;
    const int kv = head[m] - a.n_heads, vv = kv - a.n_kv_heads;
    const long long to = SCATTER && kv >= 0 ? pool_row[r[m]] : (long long)(row0 + r[m]);
    if (to < 0) continue;
    f16* dst = kv < 0               ? a.q_out + to * a.ldq_out + (size_t)head[m] * a.head_dim
               : SCATTER && vv >= 0 ? a.v_out + to * a.ldk_out + (size_t)vv * a.head_dim
                                    : a.k_out + to * a.ldk_out + (size_t)kv * a.head_dim;
    if (!moves[m]) {
      const float2* t = turns + (size_t)r[m] * half;
      if (PAIRS) turn<true>(x[m], y[m], t + 4 * i[m], t + 4 * j[m]);
      else turn<false>(x[m], y[m], t + 8 * i[m], nullptr);
    }
    st16_stream(dst + 8 * i[m], as_u4(x[m]));
    st16_stream(dst + 8 * j[m], as_u4(y[m]));
  }
}

// Any sizes, strides and alignment, in place: a pair for each thread and step.
template <bool PAIRS>
__global__ void __launch_bounds__(256) k_rotary_scalar(const RotaryArgs a) {
  extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
  float2* turns = reinterpret_cast<float2*>(smem);
  const int half = a.rotary_dim / 2;
  const int row0 = blockIdx.x * a.rows;
  const int rows = min(a.rows, a.n_rows - row0);
  for (int e = threadIdx.x; e < rows * half; e += 256)
    turns[e] = turn_of(angle_of(a, row0 + e / half, e % half));
  __syncthreads();
  const int per_row = (a.n_heads + a.n_kv_heads) * half;
  for (int e = threadIdx.x; e < rows * per_row; e += 256) {
    const int r = e / per_row, head = e % per_row / half, i = e % half;
    const size_t row = row0 + r;
    f16* x = head < a.n_heads ? a.q_out + row * a.ldq + (size_t)head * a.head_dim
                              : a.k_out + row * a.ldk + (size_t)(head - a.n_heads) * a.head_dim;
    f16 *p1 = x + (PAIRS ? 2 * i : i), *p2 = PAIRS ? p1 + 1 : p1 + half;
    const float2 c = turns[(size_t)r * half + i];
    const float x1 = (float)*p1, x2 = (float)*p2;
    *p1 = (f16)(x1 * c.x - x2 * c.y);
    *p2 = (f16)(x2 * c.x + x1 * c.y);
  }
}

// Any even rotary_dim, on the way into the cache: vectors of eight elements, of which those that turn find their
// partners by themselves: as pairs in the same vector, as halves at addresses that are no vectors', from the
// first-level cache. 2001 rows of 16 + 2 x 16 heads of 80 into the cache take 10.1 us with 20 or 40 elements turned as
// halves and 8.1 as pairs, 9.7 and 9.9 by the kernel above with all of them (floor 5.1).
template <bool PAIRS>
__global__ void __launch_bounds__(256) k_rotary_scatter_any(const RotaryArgs a) {
  extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
  float2* turns = reinterpret_cast<float2*>(smem);
  const int tid = threadIdx.x, half = a.rotary_dim / 2;
  const int row0 = blockIdx.x * a.rows, rows = min(a.rows, a.n_rows - row0);
  long long* pool_row = reinterpret_cast<long long*>(turns + (size_t)a.rows * half);
  if (tid < rows) pool_row[tid] = pool_row_of(a, row0 + tid);
  for (int e = tid; e < rows * half; e += 256) {
    const int r = (int)fdiv(e, a.by_half);
    turns[e] = turn_of(angle_of(a, row0 + r, e - r * half));
  }
  lds_barrier();
  for (int unit = tid; unit < rows * a.per_row; unit += 256) {
    const int r = (int)fdiv(unit, a.by_row), rest = unit - r * a.per_row;
    const int head = (int)fdiv(rest, a.by_unit), e0 = 8 * (rest - head * (int)a.by_unit.d);
    const int kv = head - a.n_heads, vv = kv - a.n_kv_heads;
    const size_t row = row0 + r;
    const f16* src = a.q + row * a.ldq + (size_t)head * a.head_dim;
    const long long to = kv < 0 ? (long long)row : pool_row[r];
    if (to < 0) continue;
    f16x8 x = as_h8(ld16(src + e0));
    if (vv < 0 && e0 < a.rotary_dim) {
      const float2* t = turns + (size_t)r * half;
      f16x8 y = x;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int at = e0 + e;
        if (at >= a.rotary_dim) continue;
        const bool one = PAIRS ? e % 2 == 0 : at < half;  // the first of its pair
        const f16 partner = PAIRS ? x[e ^ 1] : src[one ? at + half : at - half];
        const float2 c = t[PAIRS ? at / 2 : one ? at : at - half];
        const float mine = (float)x[e] * c.x, other = (float)partner * c.y;
        y[e] = (f16)(one ? mine - other : mine + other);
      }
      x = y;
    }
    f16* dst = kv < 0   ? a.q_out + to * a.ldq_out + (size_t)head * a.head_dim
               : vv < 0 ? a.k_out + to * a.ldk_out + (size_t)kv * a.head_dim
                        : a.v_out + to * a.ldk_out + (size_t)vv * a.head_dim;
    st16_stream(dst + e0, as_u4(x));
  }
}

// Rows of a block of k_rotary_scalar: its cosines and sines fill at most 32 KiB.
int rows_of_block(int n_rows, int half, int most) {
  int rows = 1;
  while (rows < most && (size_t)2 * rows * half * 8 <= 32768 && n_rows / (2 * rows) >= 512) rows *= 2;
  return rows;
}

// k_rotary's launch for rows of `heads` heads of `units` units each.
template <bool SCATTER>
int launch_rotary(RotaryArgs& a, int heads, int units, bool pairs, hipStream_t stream) {
  const int half = a.rotary_dim / 2;
  if ((long long)heads * units > 0x7FFFFFFF / 64) return LLMK_ERR_UNSUPPORTED;
  a.per_row = heads * units;
  // as many rows as 256 threads take (at most 8, whose page numbers and angles they load); a wide row by blocks
  // of up to 512. In place one unit a thread: four, and rows to match, took 9.5 us and not 10.4 for 4000 rows of 40
  // heads of 64, but 20.4 and not 18.2 for 8000, 5.2 and not 4.4 for 1000, 4.2 and not 2.7 for 256; between 1000 and
  // 8000 rows it is not known where they begin and cease to win.
  const auto rows_of = [&](int units_of_block) {
    int rows = units_of_block / a.per_row;
    rows = rows < 1 ? 1 : rows > 8 ? 8 : rows;
    while (rows > 1 && (size_t)rows * half * 8 > 32768) --rows;
    return rows > a.n_rows ? a.n_rows : rows;
  };
  // Three units a thread on the way into the cache where one would be 1.2 to 3 rounds of all the card's waves: 2000
  // rows of 36 heads of 128 take 10.2 us and not 11.1, 3000 13.6 and not 15.3, 3000 rows of 48 heads of 64 10.3 and
  // 11.1; but 1500 of these 7.4 and not 6.8, 8000 rows of 10 heads of 256 20.9 and 18.8, 1000 rows in place 4.2 and
  // 3.6.
  const long long all = (long long)a.n_rows * a.per_row;
  const int many = SCATTER && all >= 400000 && all < 1000000 ? 3 : 1;
  a.rows = rows_of(256 * many);
  const int units_all = a.rows * a.per_row;
  a.chunks = (int)ceil_div(units_all, 512 * many);
  const int threads = (int)ceil_div(ceil_div(ceil_div(units_all, a.chunks), many), 64) * 64;
  a.by_row = make_fastdiv((uint32_t)a.per_row);
  a.by_unit = make_fastdiv((uint32_t)units);
  a.by_half = make_fastdiv((uint32_t)half);
  const size_t blocks = (size_t)ceil_div((size_t)a.n_rows, (size_t)a.rows) * a.chunks;
  if (!grid_takes(blocks, 256)) return LLMK_ERR_UNSUPPORTED;
  const size_t lds = (size_t)a.rows * (half * 8 + (SCATTER ? 8 : 0));
  const dim3 grid((unsigned)blocks), block(threads);
  if (SCATTER && many == 3)
    return launch(pairs ? k_rotary<true, true, 3> : k_rotary<false, true, 3>, grid, block, lds, stream, a);
  return launch(pairs ? k_rotary<true, SCATTER, 1> : k_rotary<false, SCATTER, 1>, grid, block, lds, stream, a);
}

// k_rotary_scatter_any's: rows for two vectors a thread, at most 8.
int launch_any(RotaryArgs& a, bool pairs, hipStream_t stream) {
  const int half = a.rotary_dim / 2, units = a.head_dim / 8;
  const long long per_row = (a.n_heads + 2LL * a.n_kv_heads) * units;
  if (per_row > 0x7FFFFFFF / 64) return LLMK_ERR_UNSUPPORTED;
  a.per_row = (int)per_row;
  a.rows = per_row >= 512 ? 1 : per_row <= 64 ? 8 : (int)(512 / per_row);
  a.by_row = make_fastdiv((uint32_t)a.per_row);
  a.by_unit = make_fastdiv((uint32_t)units);
  a.by_half = make_fastdiv((uint32_t)half);
  const size_t blocks = ceil_div((size_t)a.n_rows, (size_t)a.rows);
  if (!grid_takes(blocks, 256)) return LLMK_ERR_UNSUPPORTED;
  return launch(pairs ? k_rotary_scatter_any<true> : k_rotary_scatter_any<false>, dim3((unsigned)blocks), dim3(256),
                (size_t)a.rows * (half * 8 + 8), stream, a);
}

int check_turn(const float* inv_freq, const int32_t* positions, int rotary_dim, int n_tables, int layout) {
  if (!inv_freq || !positions || n_tables <= 0 ||
      (layout != LLMK_ROTARY_HALVES && layout != LLMK_ROTARY_PAIRS))
    return LLMK_ERR_INVALID_VALUE;
  return rotary_dim % 2 ? LLMK_ERR_SHAPE : LLMK_OK;
}

}  // namespace
}  // namespace llmk

using namespace llmk;

extern "C" int llmk_rotary_apply(uint16_t* q, int ldq, uint16_t* k, int ldk, const int32_t* positions,
                                 const float* inv_freq, const int32_t* table_ids, const float* scales,
                                 int n_rows, int n_heads, int n_kv_heads, int head_dim, int rotary_dim,
                                 int n_tables, int layout, void* stream) {
  if (n_rows < 0 || n_heads < 0 || n_kv_heads < 0 || head_dim <= 0 || rotary_dim <= 0)
    return LLMK_ERR_INVALID_VALUE;
  if (rotary_dim > head_dim || (long long)ldq < (long long)n_heads * head_dim ||
      (long long)ldk < (long long)n_kv_heads * head_dim)
    return LLMK_ERR_SHAPE;
  if (n_rows == 0 || (n_heads == 0 && n_kv_heads == 0)) return LLMK_OK;
  if ((n_heads > 0 && !q) || (n_kv_heads > 0 && !k)) return LLMK_ERR_INVALID_VALUE;
  const int st = check_turn(inv_freq, positions, rotary_dim, n_tables, layout);
  if (st != LLMK_OK) return st;
  if (head_dim > 4096) return LLMK_ERR_UNSUPPORTED;
  const Rows turned_q{reinterpret_cast<uintptr_t>(q), n_rows, ldq, n_heads, head_dim, rotary_dim};
  const Rows turned_k{reinterpret_cast<uintptr_t>(k), n_rows, ldk, n_kv_heads, head_dim, rotary_dim};
  if (n_heads > 0 && n_kv_heads > 0 && overlap(turned_q, turned_k)) return LLMK_ERR_INVALID_VALUE;
  RotaryArgs a{};
  a.q = a.q_out = reinterpret_cast<f16*>(q);
  a.k = a.k_out = reinterpret_cast<f16*>(k);
  a.positions = positions;
  a.table_ids = table_ids;
  a.inv_freq = inv_freq;
  a.scales = scales;
  a.ldq = a.ldq_out = ldq;
  a.ldk = a.ldk_out = ldk;
  a.n_rows = n_rows;
  a.n_heads = n_heads;
  a.n_kv_heads = n_kv_heads;
  a.head_dim = head_dim;
  a.rotary_dim = rotary_dim;
  a.n_tables = n_tables;
  const bool vectors = head_dim % 8 == 0 && rotary_dim % 16 == 0 &&
                       (n_heads == 0 || (aligned16(q) && ldq % 8 == 0)) &&
                       (n_kv_heads == 0 || (aligned16(k) && ldk % 8 == 0));
  const bool pairs = layout == LLMK_ROTARY_PAIRS;
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (vectors) return launch_rotary<false>(a, n_heads + n_kv_heads, rotary_dim / 16, pairs, s);
  a.rows = rows_of_block(n_rows, rotary_dim / 2, 16);
  const unsigned blocks = ceil_div((size_t)n_rows, (size_t)a.rows);
  if (!grid_takes(blocks, 256) || (long long)a.rows * (n_heads + n_kv_heads) * head_dim > 0x7FFFFFFF - 4096)
    return LLMK_ERR_UNSUPPORTED;
  return launch(pairs ? k_rotary_scalar<true> : k_rotary_scalar<false>, dim3(blocks), dim3(256),
                (size_t)a.rows * (rotary_dim / 2) * 8, s, a);
}

extern "C" int llmk_qkv_rotary_scatter(const uint16_t* qkv, int ld, uint16_t* q_out, uint16_t* k_pool,
                                       uint16_t* v_pool, const int32_t* block_tables,
                                       const int32_t* positions, const float* inv_freq,
                                       const int32_t* table_ids, const float* scales, int n,
                                       int max_pages, int page_size, int n_heads, int n_kv_heads,
                                       int head_dim, int rotary_dim, int n_tables, int layout,
                                       void* stream) {
  if (n < 0 || max_pages <= 0 || page_size <= 0 || n_heads <= 0 || n_kv_heads <= 0 || head_dim <= 0 ||
      rotary_dim <= 0)
    return LLMK_ERR_INVALID_VALUE;
  if (head_dim % 16 || rotary_dim % 2 || rotary_dim > head_dim || (rotary_dim % 16 && head_dim % rotary_dim) || ld % 8 ||
      (long long)ld < (n_heads + 2LL * n_kv_heads) * head_dim)
    return LLMK_ERR_SHAPE;
  if (n == 0) return LLMK_OK;
  if (!qkv || !q_out || !k_pool || !v_pool || !block_tables) return LLMK_ERR_INVALID_VALUE;
  const int st = check_turn(inv_freq, positions, rotary_dim, n_tables, layout);
  if (st != LLMK_OK) return st;
  if (!aligned16(qkv) || !aligned16(q_out) || !aligned16(k_pool) || !aligned16(v_pool))
    return LLMK_ERR_ALIGNMENT;
  if (head_dim > 512) return LLMK_ERR_UNSUPPORTED;
  const size_t read = (size_t)(n - 1) * ld + ((size_t)n_heads + 2 * (size_t)n_kv_heads) * head_dim;
  if (qkv < q_out + (size_t)n * n_heads * head_dim && q_out < qkv + read) return LLMK_ERR_INVALID_VALUE;
  RotaryArgs a{};
  a.q = reinterpret_cast<const f16*>(qkv);
  a.k = a.q + (size_t)n_heads * head_dim;
  a.v = a.k + (size_t)n_kv_heads * head_dim;
  a.q_out = reinterpret_cast<f16*>(q_out);
  a.k_out = reinterpret_cast<f16*>(k_pool);
  a.v_out = reinterpret_cast<f16*>(v_pool);
  a.positions = positions;
  a.table_ids = table_ids;
  a.tables = block_tables;
  a.inv_freq = inv_freq;
  a.scales = scales;
  a.ldq = a.ldk = ld;
  a.ldq_out = n_heads * head_dim;
  a.ldk_out = n_kv_heads * head_dim;
  a.n_rows = n;
  a.n_heads = n_heads;
  a.n_kv_heads = n_kv_heads;
  a.head_dim = head_dim;
  a.rotary_dim = rotary_dim;
  a.n_tables = n_tables;
  a.max_pages = max_pages;
  a.page_size = page_size;
  const bool pairs = layout == LLMK_ROTARY_PAIRS;
  hipStream_t s = static_cast<hipStream_t>(stream);
  return rotary_dim % 16 ? launch_any(a, pairs, s)
                         : launch_rotary<true>(a, n_heads + 2 * n_kv_heads, head_dim / 16, pairs, s);
}
