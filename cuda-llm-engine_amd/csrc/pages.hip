// The pages of a cache that sequences share: copies of pages, the fork from one batch to the next with
// its counts of holders, and compaction. Integers but for the copies; nothing depends on the order in
// which blocks run: counts are added up, and every page number comes from a count of what lies in front.
#include <string.h>

#include "common.hpp"

namespace llmk {
namespace {

// ---------------------------------------------------------------------------------------------
// copies
// ---------------------------------------------------------------------------------------------
constexpr int kPools = 64;        // of a launch
constexpr int kPiece = 64 * 16 * 4;  // bytes that a wave copies at a time: 4 vectors a lane

struct CopyArgs {
  unsigned char* pool[kPools];
  size_t bytes[kPools];
  int first[kPools + 1];  // of each pool's pieces among a pair's
  const int *copies, *count;
  int n_pools, n_copies, num_pages;
};

template <bool VECTORS>
__global__ void __launch_bounds__(256) k_copy_pages(const CopyArgs a) {
  const int lane = threadIdx.x & 63;
  const int n = a.count ? min(max(*a.count, 0), a.n_copies) : a.n_copies;
  const long long pieces = a.first[a.n_pools], total = n * pieces;
  const long long step = (long long)gridDim.x * 4;
  for (long long e = (long long)blockIdx.x * 4 + (threadIdx.x >> 6); e < total; e += step) {
    const int pair = (int)(e / pieces), piece = (int)(e % pieces);
    const int from = a.copies[2 * (size_t)pair], to = a.copies[2 * (size_t)pair + 1];
    if ((unsigned)from >= (unsigned)a.num_pages || (unsigned)to >= (unsigned)a.num_pages || from == to)
      continue;
    int lo = 0, hi = a.n_pools;
    while (hi - lo > 1) {
      const int mid = (lo + hi) / 2;
      if (a.first[mid] <= piece) lo = mid; else hi = mid;
    }
    const size_t bytes = a.bytes[lo], at = (size_t)(piece - a.first[lo]) * kPiece;
    const unsigned char* src = a.pool[lo] + from * bytes;
    unsigned char* dst = a.pool[lo] + to * bytes;
    if (VECTORS) {
      u32x4 x[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const size_t o = at + (i * 64 + lane) * 16;
        if (o < bytes) x[i] = ld16_stream(src + o);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const size_t o = at + (i * 64 + lane) * 16;
        if (o < bytes) st16_stream(dst + o, x[i]);
      }
    } else {
      const size_t end = min(bytes, at + kPiece);
      for (size_t o = at + 4 * lane; o < end; o += 256)
        *reinterpret_cast<uint32_t*>(dst + o) = *reinterpret_cast<const uint32_t*>(src + o);
    }
  }
}

// ---------------------------------------------------------------------------------------------
// block-wide sums, 256 or 1024 threads
// ---------------------------------------------------------------------------------------------
__device__ __forceinline__ int wave_scan(int v) {  // inclusive
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int d = 1; d < 64; d *= 2) {
    const int o = __shfl_up(v, d);
    if (lane >= d) v += o;
  }
  return v;
}

// The sum of v over the threads in front, and *total over all. part: one int for each wave.
__device__ __forceinline__ int block_scan(int v, int* part, int* total) {
  const int wave = threadIdx.x >> 6, waves = blockDim.x >> 6;
  const int in = wave_scan(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 63) part[wave] = in;
  __syncthreads();
  int before = 0, all = 0;
  for (int w = 0; w < waves; ++w) {
    before += w < wave ? part[w] : 0;
    all += part[w];
  }
  *total = all;
  return before + in - v;
}

// ---------------------------------------------------------------------------------------------
// fork
// ---------------------------------------------------------------------------------------------
struct ForkArgs {
  const int *tables, *lens, *parents, *reserve;
  int *refs, *new_tables, *new_lens, *copies, *counts;
  int *fresh, *list;  // workspace: wanted pages of each child, then of those in front; free pages
  int n_old, n_new, max_pages, page_size, num_pages, most;
};

constexpr int kWanted = -2;  // an entry of a new table that waits for a fresh page

// How many pages the old row holds; the same in every thread of the block.
__device__ __forceinline__ int held_pages(const int* row, int max_pages, int num_pages, int* shared) {
  if (threadIdx.x == 0) *shared = max_pages;
  __syncthreads();
  int end = max_pages;
  for (int j = threadIdx.x; j < max_pages; j += blockDim.x)
    if ((unsigned)row[j] >= (unsigned)num_pages) {
      end = j;
      break;
    }
  if (end < max_pages) atomicMin(shared, end);
  __syncthreads();
  const int held = *shared;
  __syncthreads();
  return held;
}

__device__ __forceinline__ int length_of(const ForkArgs& a, int parent, int held) {
  const long long most = (long long)held * a.page_size;
  const int len = a.lens[parent];
  return len < 0 ? 0 : (int)(len < most ? len : most);
}

// The new rows, with what they keep, and how many fresh pages they want. Reads counts, changes none.
__global__ void __launch_bounds__(256) k_fork_rows(const ForkArgs a) {
  __shared__ int shared, part[4];
  const int c = blockIdx.x, p = a.parents[c];
  const bool has = (unsigned)p < (unsigned)a.n_old;
  const int* row = a.tables + (size_t)(has ? p : 0) * a.max_pages;
  const int held = has ? held_pages(row, a.max_pages, a.num_pages, &shared) : 0;
  const int len = has ? length_of(a, p, held) : 0;
  int elder = 0;
  for (int i = threadIdx.x; i < c; i += 256) elder |= a.parents[i] == p;
  const bool first = !__syncthreads_or(elder);
  const int room = a.reserve ? max(a.reserve[c], 0) : 0;
  const long long want = ((long long)len + room + a.page_size - 1) / a.page_size;
  const int need = (int)(want < a.max_pages ? want : a.max_pages);
  const int whole = len / a.page_size;
  int fresh = 0;
  for (int j = threadIdx.x; j < a.max_pages; j += 256) {
    int to = -1;
    if (j < whole) to = row[j];
    else if (j < need) {
      to = kWanted;
      if (first && j < held && a.refs[row[j]] == 1) to = row[j];
      fresh += to == kWanted;
    }
    a.new_tables[(size_t)c * a.max_pages + j] = to;
  }
  int total;
  block_scan(fresh, part, &total);
  if (threadIdx.x == 0) {
    a.fresh[c] = total;
    a.new_lens[c] = len;
  }
}

// The holders of the old rows' pages: each lets go once, the children take.
__global__ void __launch_bounds__(256) k_fork_refs(const ForkArgs a) {
  __shared__ int shared, children, first;
  const int p = blockIdx.x;
  const int* row = a.tables + (size_t)p * a.max_pages;
  if (threadIdx.x == 0) {
    children = 0;
    first = a.n_new;
  }
  const int held = held_pages(row, a.max_pages, a.num_pages, &shared);
  for (int c = threadIdx.x; c < a.n_new; c += 256)
    if (a.parents[c] == p) {
      atomicAdd(&children, 1);
      atomicMin(&first, c);
    }
  __syncthreads();
  const int whole = length_of(a, p, held) / a.page_size;
  for (int j = threadIdx.x; j < held; j += 256) {
    const int takes = j < whole ? children
                      : children ? a.new_tables[(size_t)first * a.max_pages + j] >= 0 : 0;
    if (takes != 1) atomicAdd(&a.refs[row[j]], takes - 1);
  }
}

// Finds the free pages that are wanted, in order, and makes them held. One block.
__global__ void __launch_bounds__(1024) k_fork_find(const ForkArgs a) {
  __shared__ int part[16];
  long long wanted = 0;
  for (int c0 = 0; c0 < a.n_new; c0 += 1024) {
    const int c = c0 + threadIdx.x, mine = c < a.n_new ? a.fresh[c] : 0;
    int total;
    const int before = block_scan(mine, part, &total);
    if (c < a.n_new) {
      const long long at = wanted + before;
      a.fresh[c] = (int)(at < a.num_pages ? at : a.num_pages);
    }
    wanted += total;
  }
  int found = 0;
  for (int p0 = 0; p0 < a.num_pages && found < wanted; p0 += 1024) {
    const int p = p0 + threadIdx.x;
    const bool free = p < a.num_pages && a.refs[p] == 0;
    int total;
    const int at = found + block_scan(free, part, &total);
    if (free && at < wanted && at < a.most) {
      a.list[at] = p;
      a.refs[p] = 1;
    }
    found += total;
  }
  if (threadIdx.x == 0) {
    const long long given = found < wanted ? found : wanted;
    a.counts[0] = (int)given;
    a.counts[1] = (int)(wanted - given);
  }
}

// Puts them into the rows.
__global__ void __launch_bounds__(256) k_fork_fill(const ForkArgs a) {
  __shared__ int part[4];
  const int c = blockIdx.x, p = a.parents[c], len = a.new_lens[c], given = a.counts[0];
  const int whole = len % a.page_size ? len / a.page_size : -1;  // the page that the length ends inside
  int base = a.fresh[c], from = -1, to = -1;
  for (int j0 = 0; j0 < a.max_pages; j0 += 256) {
    const int j = j0 + threadIdx.x;
    int* entry = a.new_tables + (size_t)c * a.max_pages + j;
    const bool waits = j < a.max_pages && *entry == kWanted;
    int total;
    const int at = base + block_scan(waits, part, &total);
    if (waits) {
      const int page = at < given ? a.list[at] : -1;
      *entry = page;
      if (j == whole && page >= 0) {
        from = a.tables[(size_t)p * a.max_pages + j];
        to = page;
      }
    }
    base += total;
  }
  if (whole < 0 ? threadIdx.x == 0 : threadIdx.x == whole % 256) {
    a.copies[2 * c] = from;
    a.copies[2 * c + 1] = to;
  }
}

// ---------------------------------------------------------------------------------------------
// compaction
// ---------------------------------------------------------------------------------------------
constexpr int kChunk = 4096;  // pages that a block looks at

struct CompactArgs {
  const int *tables, *refs;
  int *new_tables, *new_refs, *copies, *counts;
  int *live;   // workspace: held pages of each chunk,
  int *rank;   // of each page among the movers, or among the holes,
  int *moves;  // and (mover, hole, the mover's holders) by rank
  int num_pages, chunks;
  long long entries;
};

__global__ void __launch_bounds__(256) k_compact_count(const CompactArgs a) {
  __shared__ int part[4];
  int n = 0;
  for (int i = threadIdx.x; i < kChunk; i += 256) {
    const int p = blockIdx.x * kChunk + i;
    n += p < a.num_pages && a.refs[p] > 0;
  }
  int total;
  block_scan(n, part, &total);
  if (threadIdx.x == 0) a.live[blockIdx.x] = total;
}

// Held pages in all, of chunks in front of `chunk`, and in front of page `n_live`.
__device__ __forceinline__ void compact_sums(const CompactArgs& a, int chunk, int* part, int* n_live,
                                             int* before, int* low) {
  int all = 0, front = 0;
  for (int i = threadIdx.x; i < a.chunks; i += blockDim.x) {
    all += a.live[i];
    front += i < chunk ? a.live[i] : 0;
  }
  block_scan(all, part, n_live);
  block_scan(front, part, before);
  const int edge = *n_live / kChunk;  // the chunk that page n_live lies in
  int below = 0;
  for (int i = threadIdx.x; i < edge && i < a.chunks; i += blockDim.x) below += a.live[i];
  for (int p = edge * kChunk + threadIdx.x; p < *n_live; p += blockDim.x) below += a.refs[p] > 0;
  block_scan(below, part, low);
}

__global__ void __launch_bounds__(256) k_compact_rank(const CompactArgs a) {
  __shared__ int part[4];
  int n_live, before, low;
  compact_sums(a, blockIdx.x, part, &n_live, &before, &low);
  const int most = a.num_pages / 2;
  for (int i = 0; i < kChunk; i += 256) {
    const int p = blockIdx.x * kChunk + i + threadIdx.x;
    const bool held = p < a.num_pages && a.refs[p] > 0;
    int total;
    const int at = before + block_scan(held, part, &total);
    before += total;
    if (p >= a.num_pages) continue;
    int rank = -1;
    if (held && p >= n_live) rank = at - low;
    if (!held && p < n_live) rank = p - at;
    a.rank[p] = rank;
    if (rank < 0 || rank >= most) continue;
    a.moves[(held ? 0 : most) + rank] = p;
    if (held) a.moves[2 * most + rank] = a.refs[p];
  }
  if (blockIdx.x == 0 && threadIdx.x == 0) {
    a.counts[0] = n_live - low;
    a.counts[1] = n_live;
  }
}

__global__ void __launch_bounds__(256) k_compact_apply(const CompactArgs a) {
  const int most = a.num_pages / 2, moved = a.counts[0], n_live = a.counts[1];
  const long long step = (long long)gridDim.x * 256;
  const long long at = (long long)blockIdx.x * 256 + threadIdx.x;
  for (long long e = at; e < a.entries; e += step) {
    int p = a.tables[e];
    if (p >= n_live && p < a.num_pages) {
      const int rank = a.rank[p];
      if ((unsigned)rank < (unsigned)moved) p = a.moves[most + rank];
    }
    a.new_tables[e] = p;
  }
  for (long long e = at; e < a.num_pages; e += step) {
    const int rank = a.rank[e];
    int refs = 0;
    if (e < n_live) refs = (unsigned)rank < (unsigned)moved ? a.moves[2 * most + rank] : a.refs[e];
    a.new_refs[e] = refs;
  }
  for (long long e = at; e < most; e += step) {
    a.copies[2 * e] = e < moved ? a.moves[e] : -1;
    a.copies[2 * e + 1] = e < moved ? a.moves[most + e] : -1;
  }
}

}  // namespace
}  // namespace llmk

using namespace llmk;

extern "C" int llmk_kv_copy_pages(void* const* pools, const size_t* page_bytes, int n_pools,
                                  const int32_t* copies, const int32_t* count, int n_copies,
                                  int num_pages, void* stream) {
  if (n_pools < 0 || n_copies < 0 || num_pages <= 0) return LLMK_ERR_INVALID_VALUE;
  if (n_pools == 0 || n_copies == 0) return LLMK_OK;
  if (!pools || !page_bytes || !copies) return LLMK_ERR_INVALID_VALUE;
  for (int i = 0; i < n_pools; ++i) {
    if (!pools[i] || page_bytes[i] == 0) return LLMK_ERR_INVALID_VALUE;
    if (page_bytes[i] % 4) return LLMK_ERR_SHAPE;
    if (reinterpret_cast<uintptr_t>(pools[i]) % 4) return LLMK_ERR_ALIGNMENT;
    if (page_bytes[i] > ((size_t)1 << 32)) return LLMK_ERR_UNSUPPORTED;
  }
  for (int i = 0; i < n_pools;) {  // a launch takes kPools pools of one kind: whole vectors, or not
    CopyArgs a{};
    a.copies = copies;
    a.count = count;
    a.n_copies = n_copies;
    a.num_pages = num_pages;
    const auto whole = [&](int p) { return aligned16(pools[p]) && page_bytes[p] % 16 == 0; };
    const bool vectors = whole(i);
    for (; i < n_pools && a.n_pools < kPools && whole(i) == vectors; ++i) {
      const int n = a.n_pools++;
      a.pool[n] = static_cast<unsigned char*>(pools[i]);
      a.bytes[n] = page_bytes[i];
      a.first[n + 1] = a.first[n] + (int)((page_bytes[i] + kPiece - 1) / kPiece);
    }
    const size_t pieces = (size_t)n_copies * a.first[a.n_pools];
    const size_t blocks = (pieces + 3) / 4;
    const int st = launch(vectors ? k_copy_pages<true> : k_copy_pages<false>,
                          dim3((unsigned)(blocks < 8192 ? blocks : 8192)), dim3(256), 0,
                          static_cast<hipStream_t>(stream), a);
    if (st != LLMK_OK) return st;
  }
  return LLMK_OK;
}

extern "C" size_t llmk_kv_fork_workspace_ints(int n_old, int n_new, int max_pages, int num_pages) {
  if (n_old < 0 || n_new < 0 || max_pages <= 0 || num_pages <= 0) return 0;
  const size_t wanted = (size_t)n_new * (size_t)max_pages;
  return (size_t)n_new + (wanted < (size_t)num_pages ? wanted : (size_t)num_pages) + 1;
}

extern "C" int llmk_kv_fork(const int32_t* block_tables, const int32_t* seq_lens,
                            const int32_t* parents, const int32_t* reserve, int32_t* refs,
                            int32_t* new_tables, int32_t* new_lens, int32_t* copies, int32_t* counts,
                            int32_t* workspace, int n_old, int n_new, int max_pages, int page_size,
                            int num_pages, void* stream) {
  if (n_old < 0 || n_new < 0 || max_pages <= 0 || page_size <= 0 || num_pages <= 0)
    return LLMK_ERR_INVALID_VALUE;
  if (!refs || !counts || !workspace || (n_old > 0 && (!block_tables || !seq_lens)) ||
      (n_new > 0 && (!parents || !new_tables || !new_lens || !copies)))
    return LLMK_ERR_INVALID_VALUE;
  if (n_old > 65535 || n_new > 65535 || max_pages > (1 << 24)) return LLMK_ERR_UNSUPPORTED;
  hipStream_t s = static_cast<hipStream_t>(stream);
  ForkArgs a{};
  a.tables = block_tables;
  a.lens = seq_lens;
  a.parents = parents;
  a.reserve = reserve;
  a.refs = refs;
  a.new_tables = new_tables;
  a.new_lens = new_lens;
  a.copies = copies;
  a.counts = counts;
  a.fresh = workspace;
  a.list = workspace + n_new;
  a.n_old = n_old;
  a.n_new = n_new;
  a.max_pages = max_pages;
  a.page_size = page_size;
  a.num_pages = num_pages;
  a.most = (int)(llmk_kv_fork_workspace_ints(n_old, n_new, max_pages, num_pages) - n_new - 1);
  int st = LLMK_OK;
  if (n_new > 0) st = launch(k_fork_rows, dim3(n_new), dim3(256), 0, s, a);
  if (st == LLMK_OK && n_old > 0) st = launch(k_fork_refs, dim3(n_old), dim3(256), 0, s, a);
  if (st == LLMK_OK) st = launch(k_fork_find, dim3(1), dim3(1024), 0, s, a);
  if (st == LLMK_OK && n_new > 0) st = launch(k_fork_fill, dim3(n_new), dim3(256), 0, s, a);
  return st;
}

extern "C" size_t llmk_kv_compact_workspace_ints(int num_pages) {
  if (num_pages <= 0) return 0;
  return (size_t)ceil_div(num_pages, kChunk) + num_pages + 3 * (size_t)(num_pages / 2);
}

extern "C" int llmk_kv_compact(const int32_t* block_tables, const int32_t* refs, int32_t* new_tables,
                               int32_t* new_refs, int32_t* copies, int32_t* counts,
                               int32_t* workspace, int n_seqs, int max_pages, int num_pages,
                               void* stream) {
  if (n_seqs < 0 || max_pages <= 0 || num_pages <= 0) return LLMK_ERR_INVALID_VALUE;
  if (!refs || !new_refs || !counts || !workspace || (num_pages > 1 && !copies) ||
      (n_seqs > 0 && (!block_tables || !new_tables)))
    return LLMK_ERR_INVALID_VALUE;
  if (num_pages > (1 << 24)) return LLMK_ERR_UNSUPPORTED;
  hipStream_t s = static_cast<hipStream_t>(stream);
  CompactArgs a{};
  a.tables = block_tables;
  a.refs = refs;
  a.new_tables = new_tables;
  a.new_refs = new_refs;
  a.copies = copies;
  a.counts = counts;
  a.chunks = (int)ceil_div(num_pages, kChunk);
  a.live = workspace;
  a.rank = workspace + a.chunks;
  a.moves = a.rank + num_pages;
  a.num_pages = num_pages;
  a.entries = (long long)n_seqs * max_pages;
  int st = launch(k_compact_count, dim3(a.chunks), dim3(256), 0, s, a);
  if (st == LLMK_OK) st = launch(k_compact_rank, dim3(a.chunks), dim3(256), 0, s, a);
  if (st != LLMK_OK) return st;
  const long long most = a.entries > num_pages ? a.entries : num_pages;
  const long long blocks = (most + 255) / 256;
  return launch(k_compact_apply, dim3((unsigned)(blocks < 2048 ? blocks : 2048)), dim3(256), 0, s, a);
}
