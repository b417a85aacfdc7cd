// Low-rank adapters of a batch's sequences beside a shared projection:
//   y[r, :] += scale_a B_a (A_a x[r, :]), a the adapter of row r's sequence.
#include "kv8.hpp"

namespace llmk {
namespace {

constexpr int kParts = 8, kMaxRank = 256;

struct LoraArgs {
  const f16 *x, *a, *b;
  const int *ranks, *ids, *starts;
  const float* scales;
  f16* y;
  int part_end[kParts];
  int ldx, ldy, n_parts, n_rows, n_seqs, n_adapters, max_rank, in;
};

// A block for each row.
__global__ void __launch_bounds__(256) k_lora_row(const LoraArgs g) {
  __shared__ float h[kParts * kMaxRank];
  const int row = blockIdx.x, wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const int s = kv8::find_seq(g.starts, g.n_seqs, row);
  if (s < 0) return;
  const int a = g.ids[s];
  if ((unsigned)a >= (unsigned)g.n_adapters) return;
  const int rank = g.ranks ? min(g.ranks[a], g.max_rank) : g.max_rank;
  if (rank <= 0) return;
  for (int t = wave; t < g.n_parts * rank; t += 4) {
    const int p = t / rank, j = t % rank;
    const f16* w = g.a + (((size_t)a * g.n_parts + p) * g.max_rank + j) * g.in;
    float sum = 0.f;
    for (int i = lane * 8; i < g.in; i += 512) {
      const f16x8 u = as_h8(ld16(g.x + (size_t)row * g.ldx + i)), v = as_h8(ld16(w + i));
#pragma unroll
      for (int e = 0; e < 8; ++e) sum += (float)u[e] * (float)v[e];
    }
    sum = wave_sum(sum);
    if (lane == 0) h[p * kMaxRank + j] = sum;
  }
  __syncthreads();
  const float scale = g.scales ? g.scales[a] : 1.f;
  const int out = g.part_end[g.n_parts - 1];
  for (int n = threadIdx.x; n < out; n += 256) {
    int p = 0;
    while (n >= g.part_end[p]) ++p;
    const f16* w = g.b + ((size_t)a * out + n) * g.max_rank;
    float sum = 0.f;
    for (int j = 0; j < rank; ++j) sum += h[p * kMaxRank + j] * (float)w[j];
    f16* y = g.y + (size_t)row * g.ldy + n;
    *y = (f16)((float)*y + scale * sum);
  }
}

}  // namespace
}  // namespace llmk

using namespace llmk;

extern "C" size_t llmk_lora_add_workspace_floats(int n_rows, int n_seqs, int n_adapters, int max_rank,
                                                 int in_features, int n_parts) {
  if (n_rows <= 0 || n_seqs <= 0 || n_adapters <= 0 || max_rank <= 0 || in_features <= 0 ||
      n_parts <= 0)
    return 0;
  return 4;
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
    if (part_ends[p] <= (p ? part_ends[p - 1] : 0)) return LLMK_ERR_INVALID_VALUE;
    if (part_ends[p] % 8) return LLMK_ERR_SHAPE;
    g.part_end[p] = part_ends[p];
  }
  if (in_features % 8 || max_rank % 8 || ldx % 8 || ldy % 8 || ldx < in_features ||
      ldy < part_ends[n_parts - 1])
    return LLMK_ERR_SHAPE;
  if (max_rank > kMaxRank || n_rows > (1 << 20) || n_seqs > (1 << 20)) return LLMK_ERR_UNSUPPORTED;
  if (n_rows == 0 || n_seqs == 0 || n_adapters == 0) return LLMK_OK;
  if (!x || !a || !b || !adapter_ids || !y || !workspace) return LLMK_ERR_INVALID_VALUE;
  if (!aligned16(x) || !aligned16(a) || !aligned16(b) || !aligned16(y) || !aligned16(workspace))
    return LLMK_ERR_ALIGNMENT;
  g.x = reinterpret_cast<const f16*>(x);
  g.a = reinterpret_cast<const f16*>(a);
  g.b = reinterpret_cast<const f16*>(b);
  g.ranks = ranks;
  g.ids = adapter_ids;
  g.starts = row_starts;
  g.scales = scales;
  g.y = reinterpret_cast<f16*>(y);
  g.ldx = ldx;
  g.ldy = ldy;
  g.n_parts = n_parts;
  g.n_rows = n_rows;
  g.n_seqs = n_seqs;
  g.n_adapters = n_adapters;
  g.max_rank = max_rank;
  g.in = in_features;
  return launch(k_lora_row, dim3(n_rows), dim3(256), 0, static_cast<hipStream_t>(stream), g);
}
