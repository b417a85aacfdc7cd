// Verification of drafted tokens against the target model's probabilities, from random numbers that
// the caller gives (speculative decoding). Row i of the c rows of a sequence holds the target's
// logits behind its first i drafts; its draft d = drafts[row] came from the distribution q of the
// draft model (its logits at the same row, or certainty where there are none):
//   p = softmax(l / t), q = softmax(l_draft / t)
//   the drafts are accepted in order while u q(d) < p(d), that is with probability min(1, p / q);
//   the first refused row gives a token of max(p - q, 0) (of p where that is 0 everywhere), and the
//   last row, which has no draft, one of p: the lowest v with w_0 + .. + w_v > u2 * total.
// So the tokens are distributed as if the target had drawn each by itself. t <= 0 (or NaN) is the
// greedy choice: a draft is accepted where it is the row's argmax, which is also the token. NaN
// logits count as -inf; where +inf occurs, its places share all probability.
//
// Which token a random number falls on is settled at the borders of sums over 10^5 weights: what
// that depends on, the row where a sequence ends, is done in 64 bits (exponentials, sums,
// comparisons). Whether a draft stands compares two numbers: there the sums are 32-bit first, off
// by less than 2^-16, and only a draft that is nearer than 2^-14 to the border has its rows summed
// again, by the one wave that judges it (exact_sum), and the launches behind wait for that: 0.5 ms
// at 128256 logits and a draft model's (64 x 5 rows with one such draft 569 us, with 8 of them 582,
// with one in each sequence 1652; 1 x 5 rows of 32000 logits 78 and not 12.6). A judged draft is
// that near with a probability of 2^-13 at most, so one call in a hundred of 64 x 5 rows holds one.
//
// Launches, none of which needs an order inside itself:
//  1. every row (target and draft) in chunks of 2048 logits, a wave each: maximum, its place where
//     the choice is greedy, sum of weights relative to the chunk's maximum. A chunk is read once and
//     kept in registers for the sum. (Chunks of a block, with barriers: 62.4 us in all below, not
//     61.0; 2 or 4 chunks of a wave one behind the other, the next one's loads ahead, 65.)
//  2. where each sequence ends, found from 1 by each of its blocks, or in a launch of its own; the
//     sums of that row, in pieces of 4096.
//  3. with draft logits: the sums of max(p - q, 0) over the row's pieces.
//  4. one block for each sequence: the piece that u2 falls into, the token in it, the outputs.
//
// What bounds it: 1 reads 2 bytes a logit (64 sequences of 5 rows, 128256 logits and a draft
// model's: 30 us for 148 MB), 2 and 3 are 64-bit exponentials, some 19 instructions each, two for
// each logit of 64 rows and twice (14 and 12 us), where sequences end takes 5 and 4 another 5.5;
// 61.4 us in all. Greedy, where 2 and 3 leave at once, 32.4. Sampling without drafts reads every
// row twice and sums it in 64 bits: 256 rows 48.6 us, 64 rows 21.1, one 10.6. A single sequence is
// launches in a row: 5 rows of 32000 logits 12.6 us, of which 3.5, 6 and 3.5 in the kernels.
#include <math.h>

#include "common.hpp"
#include "verify_end.hpp"

namespace llmk {
namespace {

using namespace verify;

constexpr int kThreads = 256, kVectors = 4;             // 16-byte vectors per thread of a chunk
constexpr int kChunk = 64 * kVectors * 8;               // logits per chunk, a wave's
// The drawn row goes in pieces of 4096 logits: a few sequences give each SIMD more than one wave,
// and pieces with a draft model's share, twice the work, spread over the CUs.
constexpr int kPieceVectors = 2, kPiece = kThreads * kPieceVectors * 8;
constexpr int kChooseThreads = kPiece / 8;              // one vector each
constexpr double kLog2e = 1.44269504088896340736;

struct Stat {
  float max, sum;  // sum: of 2^((l - max) log2e / t)
  int at;          // the lowest place of the maximum, where the choice is greedy
  int pad;
};

constexpr float kFar = 3.0e38f;  // at most

struct VerifyArgs {
  const f16* logits;
  const f16* draft_logits;
  const int* drafts;
  const int* starts;
  const float* temperature;
  const float* accept_u;
  const float* sample_u;
  int* n_accepted;
  int* tokens;
  Stat* stats;    // [2][n_rows][chunks]: target, draft
  End* ends;      // [n_seqs]
  double2* sums;  // [n_seqs][pieces]: of the target's weights (without a refused certain draft's),
                  // and of the draft model's, or that draft's weight in its piece
  double* left;   // [n_seqs][pieces]: of max(p - q, 0)
  int n_rows, n_seqs, vocab, chunks, pieces;
};

// 2^y for y from -2^31 to 0, to 2^-40 of it: the whole part by the exponent, f of at most 1/2 by 1
// + f g(f), with the g of degree 7 whose largest error there is the least. 2^0 is 1 exactly.
__device__ __forceinline__ double exp2_64(double y) {
  const double n = __builtin_rint(y), f = y - n;
  double p = 1.31789487561122369e-06;
  p = __builtin_fma(p, f, 1.53091560970623410e-05);
  p = __builtin_fma(p, f, 1.54038254120923311e-04);
  p = __builtin_fma(p, f, 1.33334548606907984e-03);
  p = __builtin_fma(p, f, 9.61812861616447544e-03);
  p = __builtin_fma(p, f, 5.55041093526646920e-02);
  p = __builtin_fma(p, f, 2.40226506981104870e-01);
  p = __builtin_fma(p, f, 6.93147180548211450e-01);
  p = __builtin_fma(p, f, 1.0);
  return __builtin_ldexp(p, (int)n);
}

// The weight of a logit under a maximum above -inf. The distance goes to [-far, 0]: at -far it
// weighs nothing, and a NaN logit, which counts as -inf, has it (the median of a NaN and two
// numbers is the lower one). Under an infinite maximum, which stands as kFar, only its equals
// weigh, 1.
__device__ __forceinline__ double weight(float l, float max, const Scale& by) {
  const float d = l - __builtin_fminf(max, kFar);
  return exp2_64((double)__builtin_amdgcn_fmed3f(d, -by.far, 0.0f) * by.k);
}
// Below 4e-36 finite logits weigh 1 to the last bit, and -kFar still 0.
__device__ __forceinline__ Scale scale_of(float t) {
  const double k = __builtin_fmax(kLog2e / (double)t, 4.0e-36);
  return Scale{k, (float)__builtin_fmin(1.0e9 / k, (double)kFar), 0};
}

// The vectors of a row: element e of the row is element e + lead of the 16-byte aligned memory that
// holds it; vector v of it is the row's elements 8 v - lead .. + 7. Those that the row does not
// fill are read one by one; places outside the row count as -inf. Streamed loads: 64 x 5 rows with
// draft logits 67.6 -> 65.8 us, 4 x 5 rows 22.8 -> 23.5.
struct Row {
  const f16* base;
  int lead, vocab;
};
__device__ __forceinline__ Row row_of(const f16* logits, size_t row, int vocab) {
  Row r;
  r.base = logits + row * vocab;
  r.lead = (int)((reinterpret_cast<uintptr_t>(r.base) & 15u) / 2);
  r.vocab = vocab;
  return r;
}
__device__ __forceinline__ f16x8 load_vector(const Row& r, int v) {
  const int e = 8 * v - r.lead;
  if (e >= 0 && e + 8 <= r.vocab) return as_h8(ld16_stream(r.base + e));
  f16x8 x;
#pragma unroll
  for (int j = 0; j < 8; ++j)
    x[j] = e + j >= 0 && e + j < r.vocab ? r.base[e + j] : (f16)-INFINITY;
  return x;
}

// Sums in 64 bits by lane moves (as wave_sum): over each 16 lanes, over the wave, and over a block
// of WAVES waves; the same in every thread. shared: WAVES numbers.
template <int CTRL, int ROWS = 0xF>  // 0 where there is no source lane, and in rows not named
__device__ __forceinline__ double dpp_f64(double v) {
  const uint64_t b = __builtin_bit_cast(uint64_t, v);
  const uint32_t lo =
      __builtin_amdgcn_update_dpp(0, (int)(uint32_t)b, CTRL, ROWS, 0xF, ROWS == 0xF);
  const uint32_t hi =
      __builtin_amdgcn_update_dpp(0, (int)(uint32_t)(b >> 32), CTRL, ROWS, 0xF, ROWS == 0xF);
  return __builtin_bit_cast(double, ((uint64_t)hi << 32) | lo);
}
__device__ __forceinline__ double readlane_f64(double v, int lane) {
  const uint64_t b = __builtin_bit_cast(uint64_t, v);
  const uint32_t lo = __builtin_amdgcn_readlane((int)(uint32_t)b, lane);
  const uint32_t hi = __builtin_amdgcn_readlane((int)(uint32_t)(b >> 32), lane);
  return __builtin_bit_cast(double, ((uint64_t)hi << 32) | lo);
}
// The sum of the lanes up to each: within 16 lanes, then the rows in front (their last lanes', by
// row_bcast).
__device__ __forceinline__ double wave_prefix(double v) {
  v = v + dpp_f64<0x111>(v);
  v = v + dpp_f64<0x112>(v);
  v = v + dpp_f64<0x114>(v);
  v = v + dpp_f64<0x118>(v);
  v = v + dpp_f64<0x142, 0xA>(v);
  return v + dpp_f64<0x143, 0xC>(v);
}
template <int LANES>
__device__ __forceinline__ double row_sum(double v) {
  v = v + dpp_f64<0xB1>(v);
  v = v + dpp_f64<0x4E>(v);
  if constexpr (LANES >= 8) v = v + dpp_f64<0x141>(v);
  if constexpr (LANES == 16) v = v + dpp_f64<0x140>(v);
  return v;
}
__device__ __forceinline__ double wave_sum(double v) {
  v = row_sum<16>(v);
  return (readlane_f64(v, 0) + readlane_f64(v, 16)) + (readlane_f64(v, 32) + readlane_f64(v, 48));
}
template <int WAVES>
__device__ __forceinline__ double block_sum(double v, double* shared) {
  static_assert(WAVES == 4 || WAVES == 8, "4 or 8 lanes take the waves' sums");
  v = wave_sum(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) shared[threadIdx.x >> 6] = v;
  __syncthreads();
  return row_sum<WAVES>(shared[threadIdx.x & (WAVES - 1)]);
}
__device__ __forceinline__ float wave_max(float v) {
  v = __builtin_fmaxf(v, dpp_f32<0xB1>(v));
  v = __builtin_fmaxf(v, dpp_f32<0x4E>(v));
  v = __builtin_fmaxf(v, dpp_f32<0x141>(v));
  v = __builtin_fmaxf(v, dpp_f32<0x140>(v));
  return __builtin_fmaxf(__builtin_fmaxf(readlane_f32(v, 0), readlane_f32(v, 16)),
                         __builtin_fmaxf(readlane_f32(v, 32), readlane_f32(v, 48)));
}
template <int CTRL>
__device__ __forceinline__ int lower_dpp(int v) {
  return min(v, __builtin_amdgcn_update_dpp(0, v, CTRL, 0xF, 0xF, true));
}
__device__ __forceinline__ int wave_min(int v) {
  v = lower_dpp<0x140>(lower_dpp<0x141>(lower_dpp<0x4E>(lower_dpp<0xB1>(v))));
  return min(min(__builtin_amdgcn_readlane(v, 0), __builtin_amdgcn_readlane(v, 16)),
             min(__builtin_amdgcn_readlane(v, 32), __builtin_amdgcn_readlane(v, 48)));
}

__device__ __forceinline__ bool is_greedy(float t) { return !(t > 0.0f); }

// Rows [first, end) of sequence s, inside the call's whatever the array holds.
__device__ __forceinline__ void rows_of(const VerifyArgs& a, int s, int& first, int& end) {
  first = a.starts ? a.starts[s] : s;
  end = a.starts ? a.starts[s + 1] : s + 1;
  first = first < 0 ? 0 : first;
  end = end > a.n_rows ? a.n_rows : end;
}

__global__ void __launch_bounds__(kThreads) k_verify_stats(const VerifyArgs a) {
  const int lane = threadIdx.x & 63;
  const unsigned unit =
      kThreads / 64 * blockIdx.x + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int chunk = unit % a.chunks, which = unit / a.chunks;
  if (which >= (a.draft_logits ? 2 : 1) * a.n_rows) return;
  const int draft = which >= a.n_rows, row = which - draft * a.n_rows;
  const Row r = row_of(draft ? a.draft_logits : a.logits, row, a.vocab);
  // the row's sequence, found by halves: few loads, the same in every thread, in front of the
  // logits' (behind them 64 x 5 rows took 69.4 us and not 67.6)
  int s = row;
  if (a.starts) {
    int lo = 0, hi = a.n_seqs + 1;
    while (hi - lo > 1) {
      const int mid = lo + (hi - lo) / 2;
      if (a.starts[mid] <= row) lo = mid; else hi = mid;
    }
    s = lo;
    if (s >= a.n_seqs || a.starts[0] > row) return;
    if (draft && row == a.starts[s + 1] - 1) return;  // no draft there
  } else if (s >= a.n_seqs) {
    return;
  }
  f16x8 x[kVectors];
#pragma unroll
  for (int j = 0; j < kVectors; ++j)
    x[j] = load_vector(r, (chunk * kVectors + j) * 64 + lane);
  const float t = a.temperature ? a.temperature[s] : 1.0f;
  const bool greedy = is_greedy(t);
  if (draft && greedy) return;
  f16x8 top = (f16x8)(f16)-INFINITY;
#pragma unroll
  for (int j = 0; j < kVectors; ++j) {
    x[j] = __builtin_elementwise_max(x[j], (f16x8)(f16)-INFINITY);  // NaN counts as -inf
    top = __builtin_elementwise_max(top, x[j]);
  }
  float best = (float)top[0];
#pragma unroll
  for (int e = 1; e < 8; ++e) best = __builtin_fmaxf(best, (float)top[e]);
  best = wave_max(best);
  float sum = 0.0f;
  int at = 0x7FFFFFFF;
  if (best > -INFINITY) {
    if (greedy) {
#pragma unroll
      for (int j = kVectors - 1; j >= 0; --j)
#pragma unroll
        for (int e = 7; e >= 0; --e)
          if ((float)x[j][e] == best)
            at = 8 * ((chunk * kVectors + j) * 64 + lane) - r.lead + e;
    } else if (best == INFINITY) {
#pragma unroll
      for (int j = 0; j < kVectors; ++j)
#pragma unroll
        for (int e = 0; e < 8; ++e) sum = sum + ((float)x[j][e] == best ? 1.0f : 0.0f);
    } else {
      // k and an exponent y are rounded, 2^-23 |y| in all and |y| <= 126 (smaller weights vanish),
      // a weight by 2^-23, 32 of them and 6 steps over lanes in a sum: less than 2^-16 of the sum.
      // k is neither 0 nor infinite, so that 0 k is 0 and -inf k is -inf.
      const float k =
          __builtin_fminf(__builtin_fmaxf((float)(kLog2e / (double)t), 1.0e-37f), 3.0e38f);
#pragma unroll
      for (int j = 0; j < kVectors; ++j)
#pragma unroll
        for (int e = 0; e < 8; ++e)
          sum = sum + __builtin_amdgcn_exp2f(((float)x[j][e] - best) * k);
    }
  }
  Stat out;
  out.max = best;
  out.sum = llmk::wave_sum(sum);
  out.at = greedy ? wave_min(at) : at;
  out.pad = 0;
  if (lane == 0) a.stats[(size_t)which * a.chunks + chunk] = out;
}

// A row's maximum, its place and its sum of weights, from its chunks; by one wave.
struct RowStat {
  float max;
  int at;
  double sum;
};
__device__ __forceinline__ RowStat row_stat(const VerifyArgs& a, size_t which, bool sums,
                                            const Scale& by) {
  const Stat* st = a.stats + which * a.chunks;
  const int lane = threadIdx.x & 63;
  float max = -INFINITY, own = -INFINITY;
  int at = 0x7FFFFFFF;
  double sum = 0.0;
  for (int c = lane; c < a.chunks; c += 64) own = __builtin_fmaxf(own, st[c].max);
  RowStat r;
  r.max = max = wave_max(own);
  for (int c = lane; c < a.chunks; c += 64) {
    const Stat x = st[c];
    if (x.max == max) at = min(at, x.at);
    if (sums && x.max > -INFINITY) sum = sum + (double)x.sum * weight(x.max, max, by);
  }
  r.at = wave_min(at);
  r.sum = sums ? wave_sum(sum) : 0.0;
  return r;
}

// A row's sum of weights in 64 bits, by one wave.
__device__ double exact_sum(const f16* logits, size_t row, int vocab, float max,
                            const Scale& by) {
  double sum = 0.0;
  for (int v = threadIdx.x & 63; v < vocab; v += 64)
    sum = sum + weight((float)logits[row * vocab + v], max, by);
  return wave_sum(sum);
}

// Where a sequence ends, in every thread of the block. Wave w looks at rows w, w + 4, ..
__device__ __forceinline__ End find_end(const VerifyArgs& a, int s) {
  __shared__ int stop;
  const int wave = threadIdx.x >> 6;
  End z;
  rows_of(a, s, z.first, z.end);
  const float t = a.temperature ? a.temperature[s] : 1.0f;
  z.greedy = is_greedy(t);
  z.by = z.greedy ? Scale{} : scale_of(t);
  if (threadIdx.x == 0) stop = z.end - 1;
  __syncthreads();
  for (int row = z.first + wave; row < z.end - 1; row += 4) {
    const int d = a.drafts[row];
    const bool inside = d >= 0 && d < a.vocab;
    const float u = a.accept_u[row];
    const size_t at = (size_t)row * a.vocab + (inside ? d : 0);
    const float ld = (float)a.logits[at], lq = a.draft_logits ? (float)a.draft_logits[at] : 0.0f;
    const RowStat p = row_stat(a, row, !z.greedy, z.by);
    bool accept;
    if (z.greedy) {
      accept = inside && p.max > -INFINITY && d == p.at;
    } else if (!inside || !(p.max > -INFINITY)) {
      accept = false;
    } else {
      // u q(d) < p(d), as one side against the other with the sums multiplied out
      const double pw = weight(ld, p.max, z.by);
      double qw = 1.0, qs = 1.0;
      float qm = -INFINITY;
      if (a.draft_logits) {
        const RowStat q = row_stat(a, (size_t)a.n_rows + row, true, z.by);
        qm = q.max;
        qw = qm > -INFINITY ? weight(lq, qm, z.by) : 0.0;
        qs = qm > -INFINITY ? q.sum : 1.0;
      }
      double one = (double)u * (qw / qs), other = pw / p.sum;
      if (__builtin_fabs(one - other) < 6.103515625e-5 * __builtin_fmax(one, other)) {
        if (qm > -INFINITY)
          one = (double)u * (qw / exact_sum(a.draft_logits, row, a.vocab, qm, z.by));
        other = pw / exact_sum(a.logits, row, a.vocab, p.max, z.by);
      }
      accept = one < other;
    }
    if (!accept) {
      if ((threadIdx.x & 63) == 0) atomicMin(&stop, row);
      break;  // this wave's later rows lie behind it
    }
  }
  __syncthreads();
  z.row = stop;
  z.last = z.row == z.end - 1;
  z.pm = z.qm = -INFINITY;
  z.at = -1;
  if (z.row >= z.first) {
    const RowStat p = row_stat(a, z.row, false, z.by);
    z.pm = p.max;
    z.at = p.at;
    if (a.draft_logits && !z.last && !z.greedy)
      z.qm = row_stat(a, (size_t)a.n_rows + z.row, false, z.by).max;
  }
  return z;
}
// As an earlier launch found it.
__device__ __forceinline__ End end_of(const VerifyArgs& a, int s) {
  return checked(a.ends[s], s, a.starts != nullptr, a.n_rows);
}
// Whether there is a token to draw.
__device__ __forceinline__ bool draws(const End& z) {
  return z.row >= z.first && !z.greedy && z.pm > -INFINITY;
}
// A certain draft that was refused, -1 if there is none.
__device__ __forceinline__ int refused(const VerifyArgs& a, const End& z) {
  return z.last || a.draft_logits ? -1 : a.drafts[z.row];
}

// The draft row's logit at the place of each element of the target row's vector v.
__device__ __forceinline__ f16x8 draft_vector(const VerifyArgs& a, size_t row, const Row& r,
                                              int v) {
  const Row d = row_of(a.draft_logits, row, a.vocab);
  if (d.lead == r.lead) return load_vector(d, v);
  f16x8 x;
  const int e = 8 * v - r.lead;
#pragma unroll
  for (int j = 0; j < 8; ++j)
    x[j] = e + j >= 0 && e + j < r.vocab ? d.base[e + j] : (f16)-INFINITY;
  return x;
}

__global__ void __launch_bounds__(kThreads) k_verify_ends(const VerifyArgs a) {
  const End z = find_end(a, blockIdx.x);
  if (threadIdx.x == 0) a.ends[blockIdx.x] = z;
}

// Block (piece and sequence, share): share 0 sums the target's weights, share 1 the draft model's.
// FIND: where the sequence ends is found here, 4 us that few blocks spend at the same time; many
// would spend them one behind the other.
template <bool FIND>
__global__ void __launch_bounds__(kThreads) k_verify_sums(const VerifyArgs a) {
  __shared__ double shared[4];
  const int piece = blockIdx.x % a.pieces, s = blockIdx.x / a.pieces, share = blockIdx.y;
  const End z = FIND ? find_end(a, s) : end_of(a, s);
  if (FIND && piece == 0 && share == 0 && threadIdx.x == 0) a.ends[s] = z;
  if (!draws(z) || (share == 1 && !(z.qm > -INFINITY))) return;
  const Row r = row_of(a.logits, z.row, a.vocab);
  const int odd = refused(a, z), v0 = piece * kPieceVectors * kThreads + threadIdx.x;
  f16x8 x[kPieceVectors];
#pragma unroll
  for (int j = 0; j < kPieceVectors; ++j)
    x[j] = share == 0 ? load_vector(r, v0 + j * kThreads)
                      : draft_vector(a, z.row, r, v0 + j * kThreads);
  const float max = share == 0 ? z.pm : z.qm;
  double sum = 0.0, of_odd = 0.0;
  if (odd < 0) {
#pragma unroll
    for (int j = 0; j < kPieceVectors; ++j)
#pragma unroll
      for (int e = 0; e < 8; ++e) sum = sum + weight((float)x[j][e], max, z.by);
  } else {
#pragma unroll
    for (int j = 0; j < kPieceVectors; ++j)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const double w = weight((float)x[j][e], max, z.by);
        const bool is_odd = 8 * (v0 + j * kThreads) - r.lead + e == odd;
        of_odd = is_odd ? w : of_odd;
        sum = sum + (is_odd ? 0.0 : w);
      }
  }
  sum = block_sum<4>(sum, shared);
  if (odd >= 0) of_odd = block_sum<4>(of_odd, shared);
  if (threadIdx.x == 0) {
    double2* to = a.sums + (size_t)s * a.pieces + piece;
    if (share == 1) {
      to->y = sum;
    } else if (z.qm > -INFINITY) {
      to->x = sum;
    } else {
      *to = make_double2(sum, of_odd);
    }
  }
}

// What the last token is drawn from: a place's weight.
struct Left {
  float pm, qm;
  Scale by;
  double ps, qs;  // ps, qs: 1 / sums, or 1 and 0 where the draft model has no share
  int odd;           // a certain draft that was refused, -1
};
__device__ __forceinline__ double left_of(const Left& w, float l, float lq, int at) {
  const double p = weight(l, w.pm, w.by);
  if (at == w.odd) return 0.0;
  return w.qs == 0.0 ? p : __builtin_fmax(p * w.ps - weight(lq, w.qm, w.by) * w.qs, 0.0);
}
// By each wave for itself, 64 pieces at a time, without a barrier; first: the sums of piece `lane`,
// 0 where there is none.
__device__ __forceinline__ Left left_from(const VerifyArgs& a, const End& z, int s, double2 first) {
  Left w = {z.pm, z.qm, z.by, 1.0, 0.0, refused(a, z)};
  if (z.qm > -INFINITY) {
    double p = first.x, q = first.y;
    for (int c = (threadIdx.x & 63) + 64; c < a.pieces; c += 64) {
      const double2 x = a.sums[(size_t)s * a.pieces + c];
      p = p + x.x;
      q = q + x.y;
    }
    w.ps = 1.0 / wave_sum(p);
    w.qs = 1.0 / wave_sum(q);
  }
  return w;
}

__global__ void __launch_bounds__(kThreads) k_verify_left(const VerifyArgs a) {
  __shared__ double shared[4];
  const int piece = blockIdx.x % a.pieces, s = blockIdx.x / a.pieces, lane = threadIdx.x & 63;
  const End z = end_of(a, s);
  const double2 first =
      lane < a.pieces ? a.sums[(size_t)s * a.pieces + lane] : make_double2(0.0, 0.0);
  if (!draws(z) || !(z.qm > -INFINITY)) return;
  const Row r = row_of(a.logits, z.row, a.vocab);
  const int v0 = piece * kPieceVectors * kThreads + threadIdx.x;
  f16x8 x[kPieceVectors], y[kPieceVectors];
#pragma unroll
  for (int j = 0; j < kPieceVectors; ++j) {
    x[j] = load_vector(r, v0 + j * kThreads);
    y[j] = draft_vector(a, z.row, r, v0 + j * kThreads);
  }
  const Left w = left_from(a, z, s, first);
  double sum = 0.0;
#pragma unroll
  for (int j = 0; j < kPieceVectors; ++j)
#pragma unroll
    for (int e = 0; e < 8; ++e)  // as left_of where the draft model has a share, no branches
      sum = sum + __builtin_fmax(weight((float)x[j][e], w.pm, w.by) * w.ps -
                                     weight((float)y[j][e], w.qm, w.by) * w.qs,
                                 0.0);
  sum = block_sum<4>(sum, shared);
  if (threadIdx.x == 0) a.left[(size_t)s * a.pieces + piece] = sum;
}

__global__ void __launch_bounds__(kChooseThreads) k_verify_choose(const VerifyArgs a) {
  constexpr int WAVES = kChooseThreads / 64;
  __shared__ double shared[WAVES];
  __shared__ int first_past, last_any;
  const int s = blockIdx.x, tid = threadIdx.x, lane = tid & 63;
  const End z = end_of(a, s);
  const double2* sums = a.sums + (size_t)s * a.pieces;
  // what all this waits for, in one go
  const double2 first = lane < a.pieces ? sums[lane] : make_double2(0.0, 0.0);
  const double first_left =  // nobody's where the draft model has no share
      a.draft_logits && lane < a.pieces ? a.left[(size_t)s * a.pieces + lane] : 0.0;
  const float u = a.sample_u[s];
  for (int row = z.first + tid; row < z.end; row += kChooseThreads)
    if (row != z.row) a.tokens[row] = row < z.row ? a.drafts[row] : -1;
  if (tid == 0) {
    a.n_accepted[s] = z.end > z.first ? z.row - z.first : 0;
    if (z.end > z.first && !draws(z)) a.tokens[z.row] = z.greedy && z.pm > -INFINITY ? z.at : -1;
  }
  if (!draws(z)) return;
  if (tid == 0) {
    first_past = 0x7FFFFFFF;
    last_any = -1;
  }
  Left w = left_from(a, z, s, first);
  // Each wave looks for the piece by itself, a lane for each. Piece c's sum; with only_p of p
  // alone, where p is nowhere above q.
  const bool drafted = w.qs != 0.0, certain = w.odd >= 0;
  bool only_p = false;
  auto piece_sum = [&](int c) {
    if (c >= a.pieces) return 0.0;
    if (drafted && !only_p) return c == lane ? first_left : a.left[(size_t)s * a.pieces + c];
    const double2 x = c == lane ? first : sums[c];
    return only_p && certain ? x.x + x.y : x.x;
  };
  auto total_of = [&] {
    double sum = piece_sum(lane);
    for (int c = lane + 64; c < a.pieces; c += 64) sum = sum + piece_sum(c);
    return wave_sum(sum);
  };
  double total = total_of();
  if (!(total > 0.0)) {
    only_p = true;
    w.odd = -1;
    w.qs = 0.0;
    total = total_of();
  }
  const double aim = (double)u * total;
  // the first piece that ends past the aim, or behind them all, by rounding, the last with any
  // weight
  int chosen = 0;
  double chosen_base = 0.0, before = 0.0;
  for (int c0 = 0; c0 < a.pieces; c0 += 64) {
    const double one = piece_sum(c0 + lane), upto = wave_prefix(one), end = before + upto;
    const uint64_t any = __builtin_amdgcn_ballot_w64(one > 0.0);
    const uint64_t past = __builtin_amdgcn_ballot_w64(one > 0.0 && end > aim);
    if (any) {
      const int at = past ? __builtin_ctzll(past) : 63 - __builtin_clzll(any);
      chosen = c0 + at;
      chosen_base = readlane_f64(end - one, at);
    }
    if (past) break;
    before = before + readlane_f64(upto, 63);
  }
  const Row r = row_of(a.logits, z.row, a.vocab);
  const int v = chosen * kChooseThreads + tid;
  const f16x8 x = load_vector(r, v), y = w.qs != 0.0 ? draft_vector(a, z.row, r, v) : x;
  double each[8], own = 0.0;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    each[e] = left_of(w, (float)x[e], (float)y[e], 8 * v - r.lead + e);
    own = own + each[e];
  }
  const double upto = wave_prefix(own);
  if (lane == 63) shared[tid >> 6] = upto;
  __syncthreads();
  double c = chosen_base + (upto - own);
  for (int k = 0; k < (tid >> 6); ++k) c = c + shared[k];
  // every thread's candidate: its first place past the aim; and its last with any weight
  int token = 0x7FFFFFFF, last = -1;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    c = c + each[e];
    if (each[e] > 0.0) {
      last = 8 * v - r.lead + e;
      if (c > aim && token == 0x7FFFFFFF) token = last;
    }
  }
  // one lane of a wave: all threads at one address take 6 us
  token = wave_min(token);
  last = -wave_min(-last);
  if (lane == 0) {
    atomicMin(&first_past, token);
    atomicMax(&last_any, last);
  }
  __syncthreads();
  if (tid == 0) a.tokens[z.row] = first_past != 0x7FFFFFFF ? first_past : last_any;
}

// No rows at all: no draft stands.
__global__ void __launch_bounds__(kThreads) k_verify_none(int* n_accepted, int n_seqs) {
  const int s = blockIdx.x * kThreads + threadIdx.x;
  if (s < n_seqs) n_accepted[s] = 0;
}

// Chunks and pieces of a row, wherever its first element lies in a vector.
int chunks_of(int vocab) { return (int)(((long long)vocab + 7 + kChunk - 1) / kChunk); }
int pieces_of(int vocab) { return (int)(((long long)vocab + 7 + kPiece - 1) / kPiece); }

}  // namespace
}  // namespace llmk

using namespace llmk;

extern "C" size_t llmk_verify_drafts_workspace_floats(int n_rows, int n_seqs, int vocab) {
  if (n_rows <= 0 || n_seqs <= 0 || vocab <= 0) return 0;
  return (size_t)n_seqs * (sizeof(End) / 4) +
         (size_t)chunks_of(vocab) * 2 * (size_t)n_rows * (sizeof(Stat) / 4) +
         (size_t)pieces_of(vocab) * (size_t)n_seqs * 6;
}

extern "C" int llmk_verify_drafts(const uint16_t* logits, const uint16_t* draft_logits,
                                  const int32_t* drafts, const int32_t* row_starts,
                                  const float* temperature, const float* accept_u,
                                  const float* sample_u, int32_t* n_accepted, int32_t* tokens,
                                  float* workspace, int n_rows, int n_seqs, int vocab,
                                  void* stream) {
  if (n_rows < 0 || n_seqs < 0 || vocab <= 0) return LLMK_ERR_INVALID_VALUE;
  if (!row_starts && n_rows != n_seqs) return LLMK_ERR_INVALID_VALUE;
  if (n_seqs == 0) return LLMK_OK;
  if (!n_accepted) return LLMK_ERR_INVALID_VALUE;
  if (n_rows > 0 && (!logits || !tokens || !workspace || !sample_u ||
                     (row_starts && (!drafts || !accept_u))))
    return LLMK_ERR_INVALID_VALUE;
  if (!aligned16(workspace)) return LLMK_ERR_ALIGNMENT;
  const int chunks = chunks_of(vocab), pieces = pieces_of(vocab);
  if ((long long)chunks * 2 * n_rows > 0x7FFFFFFFLL || (long long)pieces * n_seqs > 0x7FFFFFFFLL ||
      vocab > 0x7FFFFFFF - 2 * kChunk)
    return LLMK_ERR_UNSUPPORTED;
  const bool drafted = row_starts && draft_logits;
  const size_t units = (size_t)chunks * (size_t)n_rows * (drafted ? 2 : 1);
  if (n_rows > 0 && (!grid_takes((units + kThreads / 64 - 1) / (kThreads / 64), kThreads) ||
                     !grid_takes((size_t)pieces * (size_t)n_seqs, kThreads) ||
                     !grid_takes((size_t)n_seqs, kChooseThreads)))
    return LLMK_ERR_UNSUPPORTED;
  VerifyArgs a;
  a.logits = reinterpret_cast<const f16*>(logits);
  a.draft_logits = drafted ? reinterpret_cast<const f16*>(draft_logits) : nullptr;
  a.drafts = drafts;
  a.starts = row_starts;
  a.temperature = temperature;
  a.accept_u = accept_u;
  a.sample_u = sample_u;
  a.n_accepted = n_accepted;
  a.tokens = tokens;
  a.stats = reinterpret_cast<Stat*>(workspace);
  a.sums = reinterpret_cast<double2*>(a.stats + (size_t)2 * n_rows * chunks);
  a.left = reinterpret_cast<double*>(a.sums + (size_t)n_seqs * pieces);
  a.ends = reinterpret_cast<End*>(a.left + (size_t)n_seqs * pieces);
  a.n_rows = n_rows;
  a.n_seqs = n_seqs;
  a.vocab = vocab;
  a.chunks = chunks;
  a.pieces = pieces;
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (n_rows == 0)
    return launch(k_verify_none, dim3(ceil_div((size_t)n_seqs, kThreads)), dim3(kThreads), 0, st,
                  n_accepted, n_seqs);
  int rc = launch(k_verify_stats, dim3(ceil_div(units, kThreads / 64)), dim3(kThreads), 0, st, a);
  const unsigned per_piece = (unsigned)pieces * (unsigned)n_seqs;
  const dim3 shares(per_piece, a.draft_logits ? 2 : 1);
  // Blocks of the drawn rows' sums up to which they find the ends themselves. 5 rows a sequence,
  // 128256 logits, draft logits, us in all without / with a launch for the ends: 4 sequences 23.2 /
  // 25.1, 8 27.6 / 29.4, 16 35.3 / 35.8, 64 80.6 / 72.1.
  constexpr unsigned kFindBlocks = 1024;
  if (rc == LLMK_OK && shares.x * shares.y <= kFindBlocks) {
    rc = launch(k_verify_sums<true>, shares, dim3(kThreads), 0, st, a);
  } else if (rc == LLMK_OK) {
    rc = launch(k_verify_ends, dim3((unsigned)n_seqs), dim3(kThreads), 0, st, a);
    if (rc == LLMK_OK) rc = launch(k_verify_sums<false>, shares, dim3(kThreads), 0, st, a);
  }
  if (rc == LLMK_OK && a.draft_logits)
    rc = launch(k_verify_left, dim3(per_piece), dim3(kThreads), 0, st, a);
  if (rc != LLMK_OK) return rc;
  return launch(k_verify_choose, dim3((unsigned)n_seqs), dim3(kChooseThreads), 0, st, a);
}
