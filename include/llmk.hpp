// llmk.hpp - the reference engine's C++ operator API on top of libllmk's C-ABI.
//
// Each function below has the name, argument list and argument meaning of the reference
// launcher it replaces (ref: kernels/*.cuh of JayeshNikam36/cuda-llm-engine), with
// cudaStream_t -> hipStream_t (default: the null stream) and __half from <hip/hip_fp16.h>.
// Including this header in place of the reference's kernels/*.cuh lets engine code such as
// ref: engine/batched.cu:44-72 call the MI355X kernels unchanged.
//
// Error behaviour follows the reference: launchers return void; a launch error is left in
// HIP's last-error state for the caller's hipGetLastError() (ref: engine/batched.cu:118); a
// violated precondition (hidden % 8, kvdim % 8, 16-byte alignment) is a fatal host error,
// printed to stderr followed by exit(1), like the reference's CUDA_CHECK (ref: engine/util.h:8-10).
// A zero-sized call is a no-op.
#pragma once

#include <hip/hip_fp16.h>
#include <hip/hip_runtime.h>

#include <cstdio>
#include <cstdlib>
#include <vector>

#include "llmk.h"

namespace llmk_shim {
inline void check(int status, const char* fn) {
  if (status >= LLMK_ERR_INVALID_VALUE && status <= LLMK_ERR_UNSUPPORTED) {
    std::fprintf(stderr, "%s: %s\n", fn, llmk_error_string(status));
    std::exit(1);
  }
}
inline uint16_t* h(__half* p) { return reinterpret_cast<uint16_t*>(p); }
inline const uint16_t* h(const __half* p) { return reinterpret_cast<const uint16_t*>(p); }
}  // namespace llmk_shim

// ref: kernels/embedding.cuh:6-7
inline void embedding_lookup(const __half* table, const int* ids, __half* out, int n_tokens,
                             int hidden, hipStream_t stream = 0) {
  llmk_shim::check(llmk_embedding_lookup(llmk_shim::h(table), ids, llmk_shim::h(out), n_tokens,
                                         hidden, stream),
                   "embedding_lookup");
}

// ref: kernels/rmsnorm.cuh:6-7
inline void rmsnorm(const __half* x, const __half* w, __half* out, int n_rows, int hidden,
                    float eps, hipStream_t stream = 0) {
  llmk_shim::check(llmk_rmsnorm(llmk_shim::h(x), llmk_shim::h(w), llmk_shim::h(out), n_rows,
                                hidden, eps, stream),
                   "rmsnorm");
}

// ref: kernels/residual_add.cuh:6
inline void residual_add(const __half* a, const __half* b, __half* out, size_t n,
                         hipStream_t stream = 0) {
  llmk_shim::check(
      llmk_residual_add(llmk_shim::h(a), llmk_shim::h(b), llmk_shim::h(out), n, stream),
      "residual_add");
}

// New fused entry point: residual_add(residual, x, residual) then rmsnorm(residual, w, out).
inline void add_rmsnorm(__half* residual, const __half* x, const __half* w, __half* out,
                        int n_rows, int hidden, float eps, hipStream_t stream = 0) {
  llmk_shim::check(llmk_add_rmsnorm(llmk_shim::h(residual), llmk_shim::h(x), llmk_shim::h(w),
                                    llmk_shim::h(out), n_rows, hidden, eps, stream),
                   "add_rmsnorm");
}

// ref: kernels/rope.cuh:7-9
inline std::vector<float> compute_rope_inv_freq(int head_dim, double theta, double factor,
                                                double low_freq_factor, double high_freq_factor,
                                                double original_max_pos) {
  std::vector<float> out(head_dim > 0 ? head_dim / 2 : 0);
  llmk_shim::check(llmk_compute_rope_inv_freq(head_dim, theta, factor, low_freq_factor,
                                              high_freq_factor, original_max_pos, out.data()),
                   "compute_rope_inv_freq");
  return out;
}

// ref: kernels/rope.cuh:13-15
inline void rope_apply(__half* q, __half* k, const int* positions, const float* inv_freq,
                       int n_tokens, int n_heads, int n_kv_heads, int head_dim,
                       hipStream_t stream = 0) {
  llmk_shim::check(llmk_rope_apply(llmk_shim::h(q), llmk_shim::h(k), positions, inv_freq,
                                   n_tokens, n_heads, n_kv_heads, head_dim, stream),
                   "rope_apply");
}

// ref: kernels/swiglu.cuh:6
inline void swiglu(const __half* gate, const __half* up, __half* out, size_t n,
                   hipStream_t stream = 0) {
  llmk_shim::check(
      llmk_swiglu(llmk_shim::h(gate), llmk_shim::h(up), llmk_shim::h(out), n, stream), "swiglu");
}

// ref: kernels/kv_scatter.cuh:7-8
inline void kv_scatter(const __half* src, __half* pool, const int* block_table, int start_pos,
                       int T, int page_size, int kvdim, hipStream_t stream = 0) {
  llmk_shim::check(llmk_kv_scatter(llmk_shim::h(src), llmk_shim::h(pool), block_table, start_pos,
                                   T, page_size, kvdim, stream),
                   "kv_scatter");
}

// ref: kernels/kv_scatter.cuh:12-13
inline void kv_scatter_batch(const __half* src, __half* pool, const int* block_tables,
                             const int* positions, int n, int max_pages, int page_size,
                             int kvdim, hipStream_t stream = 0) {
  llmk_shim::check(llmk_kv_scatter_batch(llmk_shim::h(src), llmk_shim::h(pool), block_tables,
                                         positions, n, max_pages, page_size, kvdim, stream),
                   "kv_scatter_batch");
}

// New fused decode entry point: rope_apply(q, k, ...) then kv_scatter_batch of k and v, with k
// left unrotated (decode attention reads K from the pool only).
inline void rope_kv_scatter_batch(__half* q, const __half* k, const __half* v, __half* k_pool,
                                  __half* v_pool, const int* block_tables, const int* positions,
                                  const float* inv_freq, int n, int max_pages, int page_size,
                                  int n_heads, int n_kv_heads, int head_dim,
                                  hipStream_t stream = 0) {
  llmk_shim::check(
      llmk_rope_kv_scatter_batch(llmk_shim::h(q), llmk_shim::h(k), llmk_shim::h(v),
                                 llmk_shim::h(k_pool), llmk_shim::h(v_pool), block_tables,
                                 positions, inv_freq, n, max_pages, page_size, n_heads,
                                 n_kv_heads, head_dim, stream),
      "rope_kv_scatter_batch");
}

// ref: kernels/attention_decode_fast.cuh:6
inline size_t attention_decode_fast_workspace_floats(int n_seq, int n_heads, int num_splits) {
  return llmk_attention_decode_fast_workspace_floats(n_seq, n_heads, num_splits);
}

// ref: kernels/attention_decode_fast.cuh:14-18. Preconditions as the reference's (page_size 16,
// head_dim 64, n_heads == 4 * n_kv_heads): a violation is a fatal host error.
inline void attention_decode_fast(const __half* q, const __half* k_pool, const __half* v_pool,
                                  const int* block_tables, const int* seq_lens, __half* out,
                                  float* workspace, int n_seq, int max_pages, int page_size,
                                  int n_heads, int n_kv_heads, int head_dim, int num_splits,
                                  hipStream_t stream = 0) {
  llmk_shim::check(
      llmk_attention_decode_fast(llmk_shim::h(q), llmk_shim::h(k_pool), llmk_shim::h(v_pool),
                                 block_tables, seq_lens, llmk_shim::h(out), workspace, n_seq,
                                 max_pages, page_size, n_heads, n_kv_heads, head_dim,
                                 num_splits, stream),
      "attention_decode_fast");
}

// The reference's split-count rule (ref: kernels/attention_decode_fast.cuh:22-29), with the
// default target rescaled for MI355X (LLMK_ATTN_TARGET_BLOCKS).
inline int choose_num_splits(int n_seq, int n_kv_heads, int max_seq_len,
                             int target_blocks = LLMK_ATTN_TARGET_BLOCKS) {
  int splits = target_blocks / (n_seq * n_kv_heads);
  const int max_splits = (max_seq_len + 15) / 16;  // never more splits than pages
  if (splits > max_splits) splits = max_splits;
  if (splits > 32) splits = 32;  // the engine's workspace holds 32 (ref: engine/batched.cu:29)
  if (splits < 1) splits = 1;
  return splits;
}

// ref: kernels/argmax.cuh:7
inline void argmax_rows(const __half* logits, int* out, int n_rows, int vocab,
                        hipStream_t stream = 0) {
  llmk_shim::check(llmk_argmax_rows(llmk_shim::h(logits), out, n_rows, vocab, stream),
                   "argmax_rows");
}

// Serving from an 8-bit KV cache (new entry points, documented in llmk.h): pools and scales as there,
// a violated precondition is a fatal host error.
inline void kv8_append(const __half* qkv, int ld, __half* q_out, uint8_t* k_pool, float* k_scale,
                       uint8_t* v_pool, float* v_scale, const int* block_tables,
                       const int* row_starts, const int* seq_lens, const float* inv_freq, int n_rows,
                       int n_seqs, int max_pages, int page_size, int n_heads, int n_kv_heads,
                       int head_dim, hipStream_t stream = 0) {
  llmk_shim::check(
      llmk_kv8_append(llmk_shim::h(qkv), ld, llmk_shim::h(q_out), k_pool, k_scale, v_pool, v_scale,
                      block_tables, row_starts, seq_lens, inv_freq, n_rows, n_seqs, max_pages,
                      page_size, n_heads, n_kv_heads, head_dim, stream),
      "kv8_append");
}

inline void kv8_gather(const uint8_t* k_pool, const float* k_scale, const uint8_t* v_pool,
                       const float* v_scale, const int* block_tables, const int* row_starts,
                       const int* seq_lens, __half* k_out, __half* v_out, int n_rows, int n_seqs,
                       int max_pages, int page_size, int n_kv_heads, int head_dim,
                       hipStream_t stream = 0) {
  llmk_shim::check(
      llmk_kv8_gather(k_pool, k_scale, v_pool, v_scale, block_tables, row_starts, seq_lens,
                      llmk_shim::h(k_out), llmk_shim::h(v_out), n_rows, n_seqs, max_pages, page_size,
                      n_kv_heads, head_dim, stream),
      "kv8_gather");
}

inline size_t kv8_attention_workspace_floats(int head_dim) {
  return llmk_kv8_attention_workspace_floats(head_dim);
}

inline void kv8_attention(const __half* q, const uint8_t* k_pool, const float* k_scale,
                          const uint8_t* v_pool, const float* v_scale, const int* block_tables,
                          const int* row_starts, const int* seq_lens, __half* out, float* workspace,
                          int n_rows, int n_seqs, int max_rows, int max_pages, int page_size,
                          int n_heads, int n_kv_heads, int head_dim, hipStream_t stream = 0) {
  llmk_shim::check(
      llmk_kv8_attention(llmk_shim::h(q), k_pool, k_scale, v_pool, v_scale, block_tables, row_starts,
                         seq_lens, llmk_shim::h(out), workspace, n_rows, n_seqs, max_rows, max_pages,
                         page_size, n_heads, n_kv_heads, head_dim, stream),
      "kv8_attention");
}

inline size_t verify_drafts_workspace_floats(int n_rows, int n_seqs, int vocab) {
  return llmk_verify_drafts_workspace_floats(n_rows, n_seqs, vocab);
}

inline void verify_drafts(const __half* logits, const __half* draft_logits, const int* drafts,
                          const int* row_starts, const float* temperature, const float* accept_u,
                          const float* sample_u, int* n_accepted, int* tokens, float* workspace,
                          int n_rows, int n_seqs, int vocab, hipStream_t stream = 0) {
  llmk_shim::check(
      llmk_verify_drafts(llmk_shim::h(logits), llmk_shim::h(draft_logits), drafts, row_starts,
                         temperature, accept_u, sample_u, n_accepted, tokens, workspace, n_rows,
                         n_seqs, vocab, stream),
      "verify_drafts");
}

// Serving requests that are not alike (new entry points, documented in llmk.h): a violated precondition is a
// fatal host error, as above.
inline size_t lora_add_workspace_floats(int n_rows, int n_seqs, int n_adapters, int max_rank,
                                        int in_features, int n_parts) {
  return llmk_lora_add_workspace_floats(n_rows, n_seqs, n_adapters, max_rank, in_features, n_parts);
}

inline void lora_add(const __half* x, int ldx, const __half* a, const __half* b, const int* ranks,
                     const float* scales, const int* adapter_ids, const int* row_starts, __half* y,
                     int ldy, const int* part_ends, int n_parts, float* workspace, int n_rows,
                     int n_seqs, int n_adapters, int max_rank, int in_features,
                     hipStream_t stream = 0) {
  llmk_shim::check(
      llmk_lora_add(llmk_shim::h(x), ldx, llmk_shim::h(a), llmk_shim::h(b), ranks, scales, adapter_ids,
                    row_starts, llmk_shim::h(y), ldy, part_ends, n_parts, workspace, n_rows, n_seqs,
                    n_adapters, max_rank, in_features, stream),
      "lora_add");
}

inline void rotary_apply(__half* q, int ldq, __half* k, int ldk, const int* positions,
                         const float* inv_freq, const int* table_ids, const float* scales, int n_rows,
                         int n_heads, int n_kv_heads, int head_dim, int rotary_dim, int n_tables,
                         int layout, hipStream_t stream = 0) {
  llmk_shim::check(
      llmk_rotary_apply(llmk_shim::h(q), ldq, llmk_shim::h(k), ldk, positions, inv_freq, table_ids,
                        scales, n_rows, n_heads, n_kv_heads, head_dim, rotary_dim, n_tables, layout,
                        stream),
      "rotary_apply");
}

inline void qkv_rotary_scatter(const __half* qkv, int ld, __half* q_out, __half* k_pool,
                               __half* v_pool, const int* block_tables, const int* positions,
                               const float* inv_freq, const int* table_ids, const float* scales, int n,
                               int max_pages, int page_size, int n_heads, int n_kv_heads, int head_dim,
                               int rotary_dim, int n_tables, int layout, hipStream_t stream = 0) {
  llmk_shim::check(
      llmk_qkv_rotary_scatter(llmk_shim::h(qkv), ld, llmk_shim::h(q_out), llmk_shim::h(k_pool),
                              llmk_shim::h(v_pool), block_tables, positions, inv_freq, table_ids, scales,
                              n, max_pages, page_size, n_heads, n_kv_heads, head_dim, rotary_dim,
                              n_tables, layout, stream),
      "qkv_rotary_scatter");
}

inline std::vector<float> compute_rotary_inv_freq(int scaling, int rotary_dim, double theta,
                                                  double factor, double original_max_pos,
                                                  double beta_fast, double beta_slow,
                                                  float* scale = nullptr) {
  std::vector<float> out(rotary_dim > 0 ? rotary_dim / 2 : 0);
  llmk_shim::check(llmk_compute_rotary_inv_freq(scaling, rotary_dim, theta, factor, original_max_pos,
                                                beta_fast, beta_slow, out.data(), scale),
                   "compute_rotary_inv_freq");
  return out;
}

inline void kv_copy_pages(void* const* pools, const size_t* page_bytes, int n_pools,
                          const int* copies, const int* count, int n_copies, int num_pages,
                          hipStream_t stream = 0) {
  llmk_shim::check(llmk_kv_copy_pages(pools, page_bytes, n_pools, copies, count, n_copies, num_pages,
                                      stream),
                   "kv_copy_pages");
}

inline size_t kv_fork_workspace_ints(int n_old, int n_new, int max_pages, int num_pages) {
  return llmk_kv_fork_workspace_ints(n_old, n_new, max_pages, num_pages);
}

inline void kv_fork(const int* block_tables, const int* seq_lens, const int* parents,
                    const int* reserve, int* refs, int* new_tables, int* new_lens, int* copies,
                    int* counts, int* workspace, int n_old, int n_new, int max_pages, int page_size,
                    int num_pages, hipStream_t stream = 0) {
  llmk_shim::check(llmk_kv_fork(block_tables, seq_lens, parents, reserve, refs, new_tables, new_lens,
                                copies, counts, workspace, n_old, n_new, max_pages, page_size,
                                num_pages, stream),
                   "kv_fork");
}

inline size_t kv_compact_workspace_ints(int num_pages) {
  return llmk_kv_compact_workspace_ints(num_pages);
}

inline void kv_compact(const int* block_tables, const int* refs, int* new_tables, int* new_refs,
                       int* copies, int* counts, int* workspace, int n_seqs, int max_pages,
                       int num_pages, hipStream_t stream = 0) {
  llmk_shim::check(llmk_kv_compact(block_tables, refs, new_tables, new_refs, copies, counts, workspace,
                                   n_seqs, max_pages, num_pages, stream),
                   "kv_compact");
}
