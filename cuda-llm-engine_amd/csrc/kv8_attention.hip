// Attention over the 8-bit KV cache (layout: kv8.hpp): out = softmax_j(q . K_j / sqrt(head_dim)) V_j
// over the positions j up to the row's own, for rows of any number a sequence.
//
// One wave for each (row, query head): 64 positions at a time, one to a lane for the scores, then
// one dim to a lane for the sums. Scores, weights and sums in 32 bits.
#include <math.h>

#include "kv8.hpp"

namespace llmk {
namespace {

using namespace kv8;

constexpr float kLog2e = 1.44269504088896341f;

struct AttentionArgs {
  Batch batch;
  const f16* q;
  const uint8_t* k_pool;
  const float* k_scale;
  const uint8_t* v_pool;
  const float* v_scale;
  f16* out;
  int n_heads, n_kv_heads;
};

template <int HD>
__global__ void __launch_bounds__(256) k_kv8_attention_rows(const AttentionArgs a) {
  const int row = blockIdx.x, lane = threadIdx.x & 63;
  const int head = blockIdx.y * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int s = __builtin_amdgcn_readfirstlane(find_seq(a.batch.starts, a.batch.n_seqs, row));
  if (s < 0 || head >= a.n_heads) return;
  const long long back = a.batch.starts ? (long long)a.batch.starts[s + 1] - row : 1;
  long long see = a.batch.lens[s] - back + 1;  // positions that the row sees
  const long long table = (long long)a.batch.max_pages * kPage;
  see = see < table ? see : table;
  const int kvh = head / (a.n_heads / a.n_kv_heads);
  const int* pages = a.batch.tables + (size_t)s * a.batch.max_pages;
  const f16* q = a.q + ((size_t)row * a.n_heads + head) * HD;
  const float scale = 1.0f / __builtin_sqrtf((float)HD);

  float m = -INFINITY, l = 0.0f, acc[HD / 64];
  for (int d = 0; d < HD / 64; ++d) acc[d] = 0.0f;
  for (long long base = 0; base < see; base += 64) {
    const long long pos = base + lane;
    float x = -INFINITY;
    if (pos < see) {
      const size_t block = (size_t)pages[pos / kPage] * a.n_kv_heads + kvh;
      const uint8_t* k = a.k_pool + (block * kPage + pos % kPage) * HD;
      const float ks = a.k_scale[block];
      float dot = 0.0f;
      for (int v = 0; v < HD / 16; ++v) {
        const u32x4 b = ld16(k + 16 * v);
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          const f16x2 lo = from_e4m3<false>(elem(b, c), ks), hi = from_e4m3<true>(elem(b, c), ks);
          const f16* qv = q + 16 * v + 4 * c;
          dot = __builtin_fmaf((float)qv[0], (float)lo[0], dot);
          dot = __builtin_fmaf((float)qv[1], (float)lo[1], dot);
          dot = __builtin_fmaf((float)qv[2], (float)hi[0], dot);
          dot = __builtin_fmaf((float)qv[3], (float)hi[1], dot);
        }
      }
      x = dot * scale;
    }
    float top = x;  // NaN scores are passed over here and come back through their weights
    for (int d = 1; d < 64; d *= 2) top = __builtin_fmaxf(top, __shfl_xor(top, d));
    const float next = __builtin_fmaxf(m, top);
    const float ref = next == -INFINITY ? 0.0f : next;
    const float corr = __builtin_amdgcn_exp2f((m - ref) * kLog2e);
    const float p = __builtin_amdgcn_exp2f((x - ref) * kLog2e);
    m = next;
    l = l * corr + p;
    for (int d = 0; d < HD / 64; ++d) acc[d] = acc[d] * corr;
    const int n = see - base < 64 ? (int)(see - base) : 64;
    for (int j = 0; j < n; ++j) {
      const float w = __shfl(p, j);
      const size_t block = (size_t)pages[(base + j) / kPage] * a.n_kv_heads + kvh;
      const uint8_t* v = a.v_pool + (block * kPage + (base + j) % kPage) * HD;
      for (int d = 0; d < HD / 64; ++d) {
        const f16x2 y = from_e4m3<false>(v[64 * d + lane], a.v_scale[block]);
        acc[d] = __builtin_fmaf(w, (float)y[0], acc[d]);
      }
    }
  }
  for (int d = 1; d < 64; d *= 2) l = l + __shfl_xor(l, d);
  f16* out = a.out + ((size_t)row * a.n_heads + head) * HD;
  for (int d = 0; d < HD / 64; ++d) out[64 * d + lane] = see > 0 ? (f16)(acc[d] / l) : (f16)0;
}

}  // namespace
}  // namespace llmk

using namespace llmk;

extern "C" size_t llmk_kv8_attention_workspace_floats(int head_dim) {
  return head_dim == 64 || head_dim == 128 ? 4 : 0;
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
  if (n_heads > 65535) return LLMK_ERR_UNSUPPORTED;
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
  a.n_heads = n_heads;
  a.n_kv_heads = n_kv_heads;
  return launch(head_dim == 64 ? k_kv8_attention_rows<64> : k_kv8_attention_rows<128>,
                dim3((unsigned)n_rows, ceil_div((size_t)n_heads, 4)), dim3(256), 0,
                static_cast<hipStream_t>(stream), a);
}
