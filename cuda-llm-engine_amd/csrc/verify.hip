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
// Which token a random number falls on is settled at the borders of sums over 10^5 weights, so
// exponentials, sums and comparisons are in 64 bits (their vector rate here is that of 32 bits).
//
// Three launches, none of which needs another's order inside itself:
//  1. every row (target and draft) in chunks of 8192 logits: maximum, its place, sum of weights
//     relative to the chunk's maximum. A chunk is read once and kept in registers for the sum.
//  2. with draft logits: the sums of max(p - q, 0) over each chunk of the row where a sequence ends.
//  3. one block for each sequence: the chunk that u2 falls into, the token in it, the outputs.
// What decides where a sequence ends is a few loads from 1; 2 and 3 each find it for themselves.
#include <math.h>

#include "common.hpp"

namespace llmk {
namespace {

constexpr int kThreads = 256, kVectors = 4;             // 16-byte vectors per thread of a chunk
constexpr int kChunk = kThreads * kVectors * 8;         // logits per chunk
constexpr double kLog2e = 1.44269504088896340736;

struct Stat {
  double sum;  // of 2^((l - max) log2e / t) over the chunk
  float max;
  int at;  // the lowest place of the maximum
};

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
  Stat* stats;   // [2][n_rows][chunks]: target, draft
  double* left;  // [n_seqs][chunks]
  int n_rows, n_seqs, vocab, chunks;
};

// 2^y for y <= 0, to the last bits of 64: the series of e^z, |z| <= ln 2 / 2, behind the whole part.
__device__ __forceinline__ double exp2_64(double y) {
  y = __builtin_fmax(y, -1100.0);
  const double n = __builtin_rint(y);
  const double z = (y - n) * 0.69314718055994530942;
  double p = 1.0 / 479001600.0;
  p = __builtin_fma(p, z, 1.0 / 39916800.0);
  p = __builtin_fma(p, z, 1.0 / 3628800.0);
  p = __builtin_fma(p, z, 1.0 / 362880.0);
  p = __builtin_fma(p, z, 1.0 / 40320.0);
  p = __builtin_fma(p, z, 1.0 / 5040.0);
  p = __builtin_fma(p, z, 1.0 / 720.0);
  p = __builtin_fma(p, z, 1.0 / 120.0);
  p = __builtin_fma(p, z, 1.0 / 24.0);
  p = __builtin_fma(p, z, 1.0 / 6.0);
  p = __builtin_fma(p, z, 0.5);
  p = __builtin_fma(p, z, 1.0);
  p = __builtin_fma(p, z, 1.0);
  return __builtin_ldexp(p, (int)n);
}

// The weight of a logit under a maximum; k = log2e / t. Equal infinities weigh 1.
__device__ __forceinline__ double weight(float l, float max, double k) {
  const float d = l == max ? 0.0f : l - max;
  return exp2_64((double)d * k);
}

__device__ __forceinline__ float logit(f16 x) {
  const float l = (float)x;
  return l != l ? -INFINITY : l;
}

// The vectors of a row: element e of the row is element e + lead of the 16-byte aligned memory that
// holds it; vector v of it is the row's elements 8 v - lead .. + 7. Those that the row does not fill
// are read one by one; places outside the row count as -inf.
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
  if (e >= 0 && e + 8 <= r.vocab) return as_h8(ld16(r.base + e));
  f16x8 x;
#pragma unroll
  for (int j = 0; j < 8; ++j)
    x[j] = e + j >= 0 && e + j < r.vocab ? r.base[e + j] : (f16)-INFINITY;
  return x;
}

__device__ __forceinline__ double block_sum(double v, double* shared) {
  for (int d = 1; d < 64; d *= 2) v = v + __shfl_xor(v, d);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) shared[threadIdx.x >> 6] = v;
  __syncthreads();
  return (shared[0] + shared[1]) + (shared[2] + shared[3]);
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
  __shared__ double shared[4];
  __shared__ float top[4];
  __shared__ int top_at[4];
  const int tid = threadIdx.x;
  const int chunk = blockIdx.x % a.chunks, which = blockIdx.x / a.chunks;
  const int draft = which >= a.n_rows, row = which - draft * a.n_rows;
  // the row's sequence, found by halves: few, and the same in every thread
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
  } else if (draft || s >= a.n_seqs) {
    return;
  }
  const float t = a.temperature ? a.temperature[s] : 1.0f;
  if (draft && is_greedy(t)) return;
  const Row r = row_of(draft ? a.draft_logits : a.logits, row, a.vocab);
  f16x8 x[kVectors];
#pragma unroll
  for (int j = 0; j < kVectors; ++j)
    x[j] = load_vector(r, (chunk * kVectors + j) * kThreads + tid);
  float best = -INFINITY;
  int at = 0x7FFFFFFF;
#pragma unroll
  for (int j = 0; j < kVectors; ++j)
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float l = logit(x[j][e]);
      if (l > best) {
        best = l;
        at = 8 * ((chunk * kVectors + j) * kThreads + tid) - r.lead + e;
      }
    }
  for (int d = 1; d < 64; d *= 2) {
    const float ob = __shfl_xor(best, d);
    const int oa = __shfl_xor(at, d);
    const bool take = ob > best || (ob == best && oa < at);
    best = take ? ob : best;
    at = take ? oa : at;
  }
  if ((tid & 63) == 0) {
    top[tid >> 6] = best;
    top_at[tid >> 6] = at;
  }
  __syncthreads();
  best = top[0];
  at = top_at[0];
  for (int w = 1; w < 4; ++w)
    if (top[w] > best || (top[w] == best && top_at[w] < at)) {
      best = top[w];
      at = top_at[w];
    }
  double sum = 0.0;
  if (!is_greedy(t) && best > -INFINITY) {
    const double k = kLog2e / (double)t;
#pragma unroll
    for (int j = 0; j < kVectors; ++j)
#pragma unroll
      for (int e = 0; e < 8; ++e) sum = sum + weight(logit(x[j][e]), best, k);
  }
  sum = block_sum(sum, shared);
  if (tid == 0) {
    Stat out;
    out.sum = sum;
    out.max = best;
    out.at = at;
    a.stats[(size_t)which * a.chunks + chunk] = out;
  }
}

// A row's maximum, its place and its sum of weights, from its chunks; by one wave.
__device__ __forceinline__ Stat row_stat(const VerifyArgs& a, size_t which, bool sums, double k) {
  const Stat* st = a.stats + which * a.chunks;
  const int lane = threadIdx.x & 63;
  Stat r;
  r.max = -INFINITY;
  r.at = 0x7FFFFFFF;
  r.sum = 0.0;
  for (int c = lane; c < a.chunks; c += 64)
    if (st[c].max > r.max) {
      r.max = st[c].max;
      r.at = st[c].at;
    }
  for (int d = 1; d < 64; d *= 2) {
    const float om = __shfl_xor(r.max, d);
    const int oa = __shfl_xor(r.at, d);
    if (om > r.max || (om == r.max && oa < r.at)) {
      r.max = om;
      r.at = oa;
    }
  }
  if (sums)
    for (int c = lane; c < a.chunks; c += 64)
      if (st[c].max > -INFINITY) r.sum = r.sum + st[c].sum * weight(st[c].max, r.max, k);
  for (int d = 1; d < 64; d *= 2) r.sum = r.sum + __shfl_xor(r.sum, d);
  return r;
}

struct End {
  int first, end, row;  // the sequence's rows, and the one that gives its last token
  bool last;            // it stands behind all drafts
  bool greedy;
  double k;
  Stat p, q;  // q: with draft logits, and not last
};

// Where a sequence ends, in every thread of the block. Wave w looks at rows w, w + 4, ..
__device__ __forceinline__ End find_end(const VerifyArgs& a, int s) {
  __shared__ int stop;
  const int wave = threadIdx.x >> 6;
  End z;
  rows_of(a, s, z.first, z.end);
  const float t = a.temperature ? a.temperature[s] : 1.0f;
  z.greedy = is_greedy(t);
  z.k = z.greedy ? 0.0 : kLog2e / (double)t;
  if (threadIdx.x == 0) stop = z.end - 1;
  __syncthreads();
  for (int row = z.first + wave; row < z.end - 1; row += 4) {
    const Stat p = row_stat(a, row, !z.greedy, z.k);
    const int d = a.drafts[row];
    bool accept;
    if (z.greedy) {
      accept = p.max > -INFINITY && d == p.at;
    } else if (d < 0 || d >= a.vocab || !(p.max > -INFINITY)) {
      accept = false;
    } else {
      const double pd = weight(logit(a.logits[(size_t)row * a.vocab + d]), p.max, z.k) / p.sum;
      double qd = 1.0;
      if (a.draft_logits) {
        const Stat q = row_stat(a, (size_t)a.n_rows + row, true, z.k);
        qd = q.max > -INFINITY
                 ? weight(logit(a.draft_logits[(size_t)row * a.vocab + d]), q.max, z.k) / q.sum
                 : 0.0;
      }
      accept = (double)a.accept_u[row] * qd < pd;
    }
    if (!accept) {
      if ((threadIdx.x & 63) == 0) atomicMin(&stop, row);
      break;  // this wave's later rows lie behind it
    }
  }
  __syncthreads();
  z.row = stop;
  z.last = z.row == z.end - 1;
  if (z.row >= z.first) {
    z.p = row_stat(a, z.row, !z.greedy, z.k);
    if (a.draft_logits && !z.last && !z.greedy) z.q = row_stat(a, (size_t)a.n_rows + z.row, true, z.k);
  }
  return z;
}

// The weight that a place has in what the last token is drawn from.
struct Left {
  float pm, qm;
  double k, ps, qs;  // 1 / sums; qs = 0: no draft model's share
  int without;       // a certain draft that was refused, -1
};
__device__ __forceinline__ double left_of(const Left& w, float l, float ld, int at) {
  const double p = weight(l, w.pm, w.k) * w.ps;
  if (at == w.without) return 0.0;
  if (w.qs == 0.0) return p;
  return __builtin_fmax(p - weight(ld, w.qm, w.k) * w.qs, 0.0);
}
__device__ __forceinline__ Left left_from(const VerifyArgs& a, const End& z) {
  Left w;
  w.pm = z.p.max;
  w.k = z.k;
  w.ps = 1.0 / z.p.sum;
  w.qm = 0.0f;
  w.qs = 0.0;
  w.without = -1;
  if (!z.last) {
    if (!a.draft_logits) {
      w.without = a.drafts[z.row];
    } else if (z.q.max > -INFINITY) {
      w.qm = z.q.max;
      w.qs = 1.0 / z.q.sum;
    }
  }
  return w;
}

// The draft row's logit at the place of each element of the target row's vector v.
__device__ __forceinline__ f16x8 draft_vector(const VerifyArgs& a, size_t row, const Row& r, int v) {
  const Row d = row_of(a.draft_logits, row, a.vocab);
  if (d.lead == r.lead) return load_vector(d, v);
  f16x8 x;
  const int e = 8 * v - r.lead;
#pragma unroll
  for (int j = 0; j < 8; ++j)
    x[j] = e + j >= 0 && e + j < r.vocab ? d.base[e + j] : (f16)-INFINITY;
  return x;
}

__global__ void __launch_bounds__(kThreads) k_verify_left(const VerifyArgs a) {
  __shared__ double shared[4];
  const int chunk = blockIdx.x % a.chunks, s = blockIdx.x / a.chunks;
  const End z = find_end(a, s);
  if (z.row < z.first || z.last || z.greedy || !(z.p.max > -INFINITY)) return;
  const Left w = left_from(a, z);
  const Row r = row_of(a.logits, z.row, a.vocab);
  double sum = 0.0;
  for (int j = 0; j < kVectors; ++j) {
    const int v = (chunk * kVectors + j) * kThreads + threadIdx.x;
    const f16x8 x = load_vector(r, v), y = draft_vector(a, z.row, r, v);
    for (int e = 0; e < 8; ++e) {
      const int at = 8 * v - r.lead + e;
      if (at >= 0 && at < a.vocab) sum = sum + left_of(w, logit(x[e]), logit(y[e]), at);
    }
  }
  sum = block_sum(sum, shared);
  if (threadIdx.x == 0) a.left[(size_t)s * a.chunks + chunk] = sum;
}

__global__ void __launch_bounds__(kThreads) k_verify_choose(const VerifyArgs a) {
  __shared__ double shared[4], before[kThreads];
  __shared__ int first_past, last_any;
  const int s = blockIdx.x, tid = threadIdx.x;
  const End z = find_end(a, s);
  for (int row = z.first + tid; row < z.end; row += kThreads)
    a.tokens[row] = row < z.row ? a.drafts[row] : -1;
  if (z.end <= z.first) {
    if (tid == 0) a.n_accepted[s] = 0;
    return;
  }
  __syncthreads();  // the row's own -1 is in place before its token
  if (tid == 0) a.n_accepted[s] = z.row - z.first;
  if (!(z.p.max > -INFINITY)) return;  // nothing to draw from
  if (z.greedy) {
    if (tid == 0) a.tokens[z.row] = z.p.at;
    return;
  }
  Left w = left_from(a, z);
  const Row r = row_of(a.logits, z.row, a.vocab);
  // the sum over this thread's own 32 places of a chunk, which follow one another
  auto mine = [&](int chunk, double* each) {
    double sum = 0.0;
    for (int j = 0; j < kVectors; ++j) {
      const int v = (chunk * kThreads + tid) * kVectors + j;
      const f16x8 x = load_vector(r, v);
      const f16x8 y = w.qs != 0.0 ? draft_vector(a, z.row, r, v) : x;
      for (int e = 0; e < 8; ++e) {
        const int at = 8 * v - r.lead + e;
        const double l =
            at >= 0 && at < a.vocab ? left_of(w, logit(x[e]), logit(y[e]), at) : 0.0;
        if (each) each[8 * j + e] = l;
        sum = sum + l;
      }
    }
    return sum;
  };
  const Stat* st = a.stats + (size_t)z.row * a.chunks;
  auto p_sum = [&](int c) {
    return st[c].max > -INFINITY ? st[c].sum * weight(st[c].max, z.p.max, z.k) * w.ps : 0.0;
  };
  // The sum without a refused draft is taken again, not subtracted: it may be all there was.
  const int odd = w.without >= 0 && w.without < a.vocab ? (w.without + r.lead) / kChunk : -1;
  const double odd_sum = odd >= 0 ? block_sum(mine(odd, nullptr), shared) : 0.0;
  bool only_p = false;
  auto chunk_sum = [&](int c) {
    if (only_p) return p_sum(c);
    if (w.qs != 0.0) return a.left[(size_t)s * a.chunks + c];
    return c == odd ? odd_sum : p_sum(c);
  };
  double total = 0.0;
  for (int c = 0; c < a.chunks; ++c) total = total + chunk_sum(c);
  if (!(total > 0.0)) {  // p is nowhere above q
    only_p = true;
    w.without = -1;
    w.qs = 0.0;
    for (int c = 0; c < a.chunks; ++c) total = total + p_sum(c);
  }
  const double aim = (double)a.sample_u[s] * total;
  int chunk = 0;
  double base = 0.0, sum = 0.0;
  for (int c = 0; c < a.chunks; ++c) {
    const double one = chunk_sum(c);
    if (one > 0.0) {  // where rounding leaves the aim behind all: the last chunk with any weight
      chunk = c;
      base = sum;
    }
    sum = sum + one;
    if (sum > aim) break;
  }
  double each[kVectors * 8];
  const double own = mine(chunk, each);
  before[tid] = own;
  if (tid == 0) {
    first_past = 0x7FFFFFFF;
    last_any = -1;
  }
  __syncthreads();
  for (int d = 1; d < kThreads; d *= 2) {
    const double add = tid >= d ? before[tid - d] : 0.0;
    __syncthreads();
    before[tid] = before[tid] + add;
    __syncthreads();
  }
  // every thread's candidate: its first place past the aim, or behind it its last with any weight
  double c = base + (tid > 0 ? before[tid - 1] : 0.0);
  int token = -1, last = -1;
  for (int e = 0; e < kVectors * 8; ++e) {
    c = c + each[e];
    const int at = (chunk * kThreads + tid) * kVectors * 8 + e - r.lead;
    if (each[e] > 0.0) {
      last = at;
      if (token < 0 && c > aim) token = at;
    }
  }
  if (token >= 0) atomicMin(&first_past, token);
  if (last >= 0) atomicMax(&last_any, last);
  __syncthreads();
  if (tid == 0) a.tokens[z.row] = first_past != 0x7FFFFFFF ? first_past : last_any;
}

int chunks_of(int vocab) { return (int)(((long long)vocab + 7 + kChunk - 1) / kChunk); }

}  // namespace
}  // namespace llmk

using namespace llmk;

extern "C" size_t llmk_verify_drafts_workspace_floats(int n_rows, int n_seqs, int vocab) {
  if (n_rows <= 0 || n_seqs <= 0 || vocab <= 0) return 0;
  const size_t chunks = (size_t)chunks_of(vocab);
  return chunks * (2 * (size_t)n_rows * (sizeof(Stat) / 4) + 2 * (size_t)n_seqs);
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
  const int chunks = chunks_of(vocab);
  if ((long long)chunks * 2 * n_rows > 0x7FFFFFFFLL || (long long)chunks * n_seqs > 0x7FFFFFFFLL ||
      vocab > 0x7FFFFFFF - 2 * kChunk)
    return LLMK_ERR_UNSUPPORTED;
  VerifyArgs a;
  a.logits = reinterpret_cast<const f16*>(logits);
  a.draft_logits = row_starts ? reinterpret_cast<const f16*>(draft_logits) : nullptr;
  a.drafts = drafts;
  a.starts = row_starts;
  a.temperature = temperature;
  a.accept_u = accept_u;
  a.sample_u = sample_u;
  a.n_accepted = n_accepted;
  a.tokens = tokens;
  a.stats = reinterpret_cast<Stat*>(workspace);
  a.left = reinterpret_cast<double*>(a.stats + (size_t)2 * n_rows * chunks);
  a.n_rows = n_rows;
  a.n_seqs = n_seqs;
  a.vocab = vocab;
  a.chunks = chunks;
  hipStream_t st = static_cast<hipStream_t>(stream);
  int rc = LLMK_OK;
  if (n_rows > 0) {
    const unsigned rows = (unsigned)n_rows * (a.draft_logits ? 2u : 1u);
    rc = launch(k_verify_stats, dim3((unsigned)chunks * rows), dim3(kThreads), 0, st, a);
    if (rc == LLMK_OK && a.draft_logits)
      rc = launch(k_verify_left, dim3((unsigned)chunks * (unsigned)n_seqs), dim3(kThreads), 0, st,
                  a);
  }
  if (rc != LLMK_OK) return rc;
  return launch(k_verify_choose, dim3((unsigned)n_seqs), dim3(kThreads), 0, st, a);
}
