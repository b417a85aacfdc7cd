// The pages of a cache that sequences share: copies of pages, the fork from one batch to the next with
// its counts of holders, and compaction. Integers but for the copies; nothing depends on the order in
// which blocks run: counts are added up, and every page number comes from a count of what lies in front.
//
// Copies are bound by bytes, tables by loads that wait for one another. Measured (one MI355X, inputs from HBM; the
// floor is each byte once at 6 TB/s), us: the fork of 8 beams and its copies in 16 layers 9.3 (0.5), k_fork 6.4 and the
// copies 3.1; of 256 beams over an 8-bit cache 25.4 (7.2), rows 4.0, holders 3.6, pages 5.8, copies 13 (43 MB); the
// compaction of 64 sequences, half the pool free, 47.6 (37.5), 5.8 and the copies 42 (231 MB at 5.5 TB/s). Larger pools:
// a fork of 256 beams by tables of 129 pages 11.5 without its copies in 2200 pages and 12.4 in 16000, by 256 pages 14.1
// in 64000; a compaction's tables in three launches, 16000 pages of 128 sequences 12.8, 250000 of 256 15.4.
//
// Between their launches forks and compactions trust the workspace with numbers and with no address (fork_notes.hpp).
#include <limits.h>

#include "common.hpp"
#include "fork_notes.hpp"

namespace llmk {
namespace {

// ---------------------------------------------------------------------------------------------
// copies
// ---------------------------------------------------------------------------------------------
constexpr int kPools = 64;            // of a launch
constexpr int kVectors = 4, kPiece = 64 * 16 * kVectors;  // of a lane, and the bytes that a wave copies

struct CopyArgs {
  unsigned char* pool[kPools];  // n_pools of any size, then n_small whose pages are `small` bytes
  size_t bytes[kPools];
  int first[kPools + 1];  // of each pool's pieces among a pair's
  const int *copies, *count;
  int n_pools, n_small, small, n_copies, num_pages, slices;
  int each;    // pieces of every pool's page, 0 if they differ
  int across;  // whether blocks side by side are of other pairs, and not of other pieces
};

// A block for each pair and four of its pieces; pairs that are none are behind one load. Pages of few
// bytes (the scales of an 8-bit cache, 32 in each of 32 pools) are taken many pools a wave, 16 bytes a lane.
template <bool VECTORS>
__global__ void __launch_bounds__(256) k_copy_pages(const CopyArgs a) {
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int group = a.across ? a.n_copies : a.slices, far = blockIdx.x / group, near = blockIdx.x - far * group;
  const int pair = a.across ? near : far, slice = a.across ? far : near;
  if (a.count && pair >= *a.count) return;
  const int from = a.copies[2 * (size_t)pair], to = a.copies[2 * (size_t)pair + 1];
  int piece = slice * 4 + wave;
  const int pieces = a.first[a.n_pools];
  if (piece < pieces) {
    int lo = 0;
    if (a.each) {
      lo = piece / a.each;
      piece -= lo * a.each;
    } else {
      for (int hi = a.n_pools; hi - lo > 1;) {
        const int mid = (lo + hi) / 2;
        if (a.first[mid] <= piece) lo = mid; else hi = mid;
      }
      piece -= a.first[lo];
    }
    const size_t bytes = a.bytes[lo], at = (size_t)piece * kPiece;
    unsigned char* pool = a.pool[lo] + at;
    if ((unsigned)from >= (unsigned)a.num_pages || (unsigned)to >= (unsigned)a.num_pages || from == to)
      return;
    const unsigned char* src = pool + from * bytes;
    unsigned char* dst = pool + to * bytes;
    if (VECTORS && at + kPiece <= bytes) {
      u32x4 x[kVectors];
#pragma unroll
      for (int i = 0; i < kVectors; ++i) x[i] = ld16_stream(src + (i * 64 + lane) * 16);
#pragma unroll
      for (int i = 0; i < kVectors; ++i) st16_stream(dst + (i * 64 + lane) * 16, x[i]);
    } else if (VECTORS) {
      for (size_t o = lane * 16; at + o < bytes; o += 1024) st16_stream(dst + o, ld16_stream(src + o));
    } else {
      const size_t end = min(bytes - at, (size_t)kPiece);
      for (size_t o = 4 * lane; o < end; o += 256)
        *reinterpret_cast<uint32_t*>(dst + o) = *reinterpret_cast<const uint32_t*>(src + o);
    }
    return;
  }
  if ((unsigned)from >= (unsigned)a.num_pages || (unsigned)to >= (unsigned)a.num_pages || from == to)
    return;
  piece -= pieces;
  const int lanes = a.small / 16;  // of a small page; VECTORS alone has such pools
  if (!VECTORS || lanes == 0) return;
  const int mine = piece * (64 / lanes) + lane / lanes;
  if (lane / lanes < 64 / lanes && mine < a.n_small) {
    unsigned char* p = a.pool[a.n_pools + mine] + lane % lanes * 16;
    st16(p + (size_t)to * a.small, ld16(p + (size_t)from * a.small));
  }
}

// ---------------------------------------------------------------------------------------------
// block-wide sums
// ---------------------------------------------------------------------------------------------
// The sum of v over the threads in front, and *total over all. part: an int for each wave, two sets of which
// take turns, so that one barrier is enough. Over a wave in 32 bits, over the block in T's.
template <typename T>
__device__ __forceinline__ T block_scan(int v, int* part, T* total) {
  const int wave = threadIdx.x >> 6, waves = blockDim.x >> 6, in = wave_scan(v);
  if ((threadIdx.x & 63) == 63) part[wave] = in;
  __syncthreads();
  const pages::Sums<T> s = pages::sums_of<T>(part, waves, wave);
  *total = s.all;
  return s.before + in - v;
}

// ---------------------------------------------------------------------------------------------
// fork
// ---------------------------------------------------------------------------------------------
struct ForkArgs {
  const int *tables, *lens, *parents, *reserve;
  int *refs, *new_tables, *new_lens, *copies, *counts;
  int* fresh;            // workspace: wanted pages of each child, then of those in front,
  pages::Column* columns;  // and their columns
  int n_old, n_new, max_pages, page_size, num_pages;
};

constexpr int kMostPages = 1 << 30;  // k_fork_find looks at up to 8192 page numbers past the last
constexpr int kFound = 4096;  // children whose counts of wanted pages are kept in LDS
constexpr int kCopied = INT_MIN;  // holders of a page that is copied from and free behind that, while pages are given

// U entries a lane, 64 apart, on their way together; behind the end, which is past `at`, `none`.
template <int U>
__device__ __forceinline__ void load_entries(const int* from, int at, int end, int none, int (&v)[U]) {
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int u = 0; u < U; ++u) v[u] = from[min(at + 64 * u + lane, end - 1)];
#pragma unroll
  for (int u = 0; u < U; ++u) v[u] = at + 64 * u + lane < end ? v[u] : none;
}

// How many pages the old row holds, whose first entries are v. A wave's work; all lanes get it.
template <int U>
__device__ __forceinline__ int held_pages(const int* row, int max_pages, int num_pages, const int (&first)[U]) {
  for (int j = 0; j < max_pages; j += 64 * U) {
    int v[U];
    if (j == 0) {
#pragma unroll
      for (int u = 0; u < U; ++u) v[u] = first[u];
    } else {
      load_entries<U>(row, j, max_pages, -1, v);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const uint64_t m = __builtin_amdgcn_ballot_w64((unsigned)v[u] >= (unsigned)num_pages);
      if (m) return min(j + 64 * u + __builtin_ctzll(m), max_pages);
    }
  }
  return max_pages;
}

// A sequence's length, of which its pages hold at most so much.
__device__ __forceinline__ int length_of(const ForkArgs& a, int len, int held) {
  const long long most = (long long)held * a.page_size;
  return len < 0 ? 0 : (int)(len < most ? len : most);
}

constexpr int kParents = 4;  // entries of `parents` that a lane has on their way: 256 a wave

// A child's row, with what it keeps, and which columns want fresh pages. Reads counts, changes none. A wave's work.
// What is known where to find is loaded first: the parent, then its row, its length and the other parents.
template <int U>
__device__ __forceinline__ void fork_row(const ForkArgs& a, int c) {
  const int lane = threadIdx.x & 63, p = a.parents[c];
  const int room = a.reserve ? max(a.reserve[c], 0) : 0;
  const bool has = (unsigned)p < (unsigned)a.n_old;
  const int* row = a.tables + (size_t)(has ? p : 0) * a.max_pages;
  int first[U], raw = 0;
#pragma unroll
  for (int u = 0; u < U; ++u) first[u] = -1;
  if (has) {
    raw = a.lens[p];
    load_entries<U>(row, 0, a.max_pages, -1, first);
  }
  uint64_t elder = 0;
  for (int i = 0; i < c && !elder; i += 64 * kParents) {
    int v[kParents];
    load_entries<kParents>(a.parents, i, c, ~p, v);
#pragma unroll
    for (int u = 0; u < kParents; ++u) elder |= __builtin_amdgcn_ballot_w64(v[u] == p);
  }
  const int held = has ? held_pages<U>(row, a.max_pages, a.num_pages, first) : 0;
  const int len = length_of(a, raw, held);
  const long long want = ((long long)len + room + a.page_size - 1) / a.page_size;
  const int need = (int)(want < a.max_pages ? want : a.max_pages);
  const int whole = len / a.page_size;
  int fresh = 0;
  bool shared = false;
  for (int j0 = 0; j0 < a.max_pages; j0 += 64 * U) {
    int v[U], alone[U];
#pragma unroll
    for (int u = 0; u < U; ++u) v[u] = first[u];
    if (j0 > 0 && j0 < held) load_entries<U>(row, j0, held, -1, v);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int j = j0 + 64 * u + lane;
      v[u] = j < held ? v[u] : -1;
      alone[u] = !elder && j >= whole && j < held && j < need ? a.refs[v[u]] : 0;
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int j = j0 + 64 * u + lane;
      const bool keeps = j < whole || alone[u] == 1, wants = !keeps && j < need;
      if (j < a.max_pages) a.new_tables[(size_t)c * a.max_pages + j] = keeps ? v[u] : -1;
      const uint64_t m = __builtin_amdgcn_ballot_w64(wants);
      shared |= !elder && __builtin_amdgcn_ballot_w64(wants && j == whole && len % a.page_size) != 0;
      if (wants)
        a.columns[(size_t)c * a.max_pages + fresh + __builtin_popcountll(m & ((1ull << lane) - 1))] =
            pages::Column{j, j == whole && len % a.page_size ? v[u] : -1};
      fresh += __builtin_popcountll(m);
    }
  }
  if (lane == 0) {
    a.fresh[c] = fresh + (shared ? pages::kCopiesShared : 0);
    a.new_lens[c] = len;
    a.copies[2 * c] = -1;
    a.copies[2 * c + 1] = -1;
  }
}

// The holders of an old row's pages: it lets go once, its children take. A wave's work.
template <int U>
__device__ __forceinline__ void fork_refs(const ForkArgs& a, int p) {
  const int lane = threadIdx.x & 63;
  const int* row = a.tables + (size_t)p * a.max_pages;
  int start[U];
  load_entries<U>(row, 0, a.max_pages, -1, start);
  const int raw = a.lens[p];
  int children = 0, first = -1;
  for (int i = 0; i < a.n_new; i += 64 * kParents) {
    int v[kParents];
    load_entries<kParents>(a.parents, i, a.n_new, -1, v);
#pragma unroll
    for (int u = 0; u < kParents; ++u) {
      const uint64_t m = __builtin_amdgcn_ballot_w64(v[u] == p);
      if (m && first < 0) first = i + 64 * u + __builtin_ctzll(m);
      children += __builtin_popcountll(m);
    }
  }
  const int held = held_pages<U>(row, a.max_pages, a.num_pages, start);
  const int whole = length_of(a, raw, held) / a.page_size;
  const int from = children == 1 ? whole : 0;  // whole pages of an only child stay as they are
  for (int j0 = from / (64 * U) * (64 * U); j0 < held; j0 += 64 * U) {
    int v[U];
#pragma unroll
    for (int u = 0; u < U; ++u) v[u] = start[u];
    if (j0 > 0) load_entries<U>(row, j0, held, -1, v);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int j = j0 + 64 * u + lane;
      if (j < from || j >= held) continue;
      const int takes = j < whole ? children
                        : children ? a.new_tables[(size_t)first * a.max_pages + j] >= 0 : 0;
      if (takes != 1) atomicAdd(&a.refs[v[u]], takes - 1);
    }
  }
}

struct Find {  // in LDS
  int begin[kFound];   // of each child's wanted pages among all,
  int child[kFound];   // and, where no child wants two, whose the k-th is, and its column
  pages::Column column[kFound];
  int part[2][16];
  int marked, listed;
};

// The k-th wanted page: child c's, which is the last whose wanted ones begin at or before k.
__device__ __forceinline__ void fork_give(const ForkArgs& a, const Find& f, bool listed, const int* begin, int k,
                                          int page) {
  int c = 0;
  pages::Column column;
  if (listed) {
    c = f.child[k];
    column = f.column[k];
  } else {
    for (int hi = a.n_new; hi - c > 1;) {
      const int mid = (c + hi) / 2;
      if (begin[mid] <= k) c = mid; else hi = mid;
    }
    column = a.columns[(size_t)c * a.max_pages + pages::place_of(k, begin[c], a.max_pages)];
  }
  column = pages::checked(column, a.max_pages, a.num_pages);
  if (column.at >= 0) a.new_tables[(size_t)c * a.max_pages + column.at] = page;
  if (column.from >= 0) {
    a.copies[2 * c] = column.from;
    a.copies[2 * c + 1] = page;
  }
}

// Which of a thread's four pages from p0 on are free, as bits; read past the first-level cache, which may hold the
// counts from before other additions.
__device__ __forceinline__ int free_bits(const ForkArgs& a, int p0) {
  const int p = p0 + 4 * threadIdx.x;
  int bits = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    bits |= (p + i < a.num_pages &&
             __hip_atomic_load(&a.refs[p + i], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == 0)
            << i;
  return bits;
}

// Gives the free pages that are wanted, in order. One block of 1024 threads. T: for sums of wanted pages.
template <typename T>
__device__ __forceinline__ void fork_find(const ForkArgs& a, Find& f) {
  const int* begin = a.n_new <= kFound ? f.begin : a.fresh;
  if (threadIdx.x == 0) {
    f.marked = 0;
    f.listed = a.n_new <= kFound;
  }
  int free = free_bits(a, 0);
  T wanted = 0;
  int turn = 0;
  for (int c0 = 0; c0 < a.n_new; c0 += 1024) {
    const int c = c0 + threadIdx.x, noted = c < a.n_new ? a.fresh[c] : 0;
    const int mine = pages::wanted_of(noted, a.max_pages);
    const pages::Column column =  // if there is one
        c < a.n_new ? a.columns[(size_t)c * a.max_pages] : pages::Column{-1, -1};
    T total;
    const T before = block_scan(mine, f.part[turn ^= 1], &total);
    if (c < a.n_new) {
      const T at = wanted + before;
      const int b = (int)(at < a.num_pages ? at : a.num_pages);
      if (a.n_new <= kFound) f.begin[c] = b; else a.fresh[c] = b;
      if (mine == 1 && at < kFound) {  // it is if no child wants two
        f.child[at] = c;
        f.column[at] = column;
      }
      if (mine > 1) f.listed = 0;
    }
    // sequences that were cut inside a page that they share: copied from, it is nobody's fresh page
    if (noted & pages::kCopiesShared) {
      const int copied = pages::checked(column, a.max_pages, a.num_pages).from;
      const int was = copied < 0 ? 1 : atomicCAS(&a.refs[copied], 0, kCopied);
      if (was == 0 || was == kCopied) f.marked = 1;
    }
    wanted += total;
  }
  __syncthreads();
  const bool some = f.marked, listed = f.listed;
  if (some) free = free_bits(a, 0);
  int found = 0;
  for (int p0 = 0; p0 < a.num_pages && found < wanted;) {
    const int next = free_bits(a, p0 + 4096);  // on its way in good time
    int total;
    int at = found + block_scan(__builtin_popcount(free), f.part[turn ^= 1], &total);
    for (; free && at < wanted; free &= free - 1, ++at) {
      const int page = p0 + 4 * threadIdx.x + __builtin_ctz(free);
      a.refs[page] = 1;
      fork_give(a, f, listed, begin, at, page);
    }
    found += total;
    p0 += 4096;
    free = next;
  }
  if (some) {
    __syncthreads();
    for (int p = threadIdx.x; p < a.num_pages; p += 1024) atomicCAS(&a.refs[p], kCopied, 0);
  }
  if (threadIdx.x == 0) {
    const T given = found < wanted ? found : wanted;
    a.counts[0] = (int)given;
    a.counts[1] = (int)min(wanted - given, (T)INT_MAX);
  }
}

// U: how many entries of a lane are on their way at a time.
template <int U>
__global__ void __launch_bounds__(256) k_fork_rows(const ForkArgs a) {
  const int c = blockIdx.x * 4 + (threadIdx.x >> 6);
  if (c < a.n_new) fork_row<U>(a, c);
}
template <int U>
__global__ void __launch_bounds__(256) k_fork_refs(const ForkArgs a) {
  const int p = blockIdx.x * 4 + (threadIdx.x >> 6);
  if (p < a.n_old) fork_refs<U>(a, p);
}
__global__ void __launch_bounds__(1024) k_fork_find(const ForkArgs a) {
  __shared__ Find f;
  fork_find<long long>(a, f);
}
// The three of them by one block, whose batches want at most 8192 pages. Its additions to counts are complete at the
// barrier and read where they were made, so no fence of the device is needed, which takes 5 us.
__global__ void __launch_bounds__(1024) k_fork(const ForkArgs a) {
  __shared__ Find f;
  const int wave = threadIdx.x >> 6;
  for (int c = wave; c < a.n_new; c += 16) fork_row<1>(a, c);
  __syncthreads();
  for (int p = wave; p < a.n_old; p += 16) fork_refs<1>(a, p);
  __syncthreads();
  fork_find<int>(a, f);
}

// ---------------------------------------------------------------------------------------------
// compaction
// ---------------------------------------------------------------------------------------------
constexpr int kChunk = 4096;  // pages that a block of 1024 threads looks at, four a thread

struct CompactArgs {
  const int *tables, *refs;
  int *new_tables, *new_refs, *copies, *counts;
  int *live;   // workspace: held pages of each chunk,
  int *rank;   // of each page among the movers, or among the holes,
  int *moves;  // and (mover, hole, the mover's holders) by rank
  int num_pages, chunks;
  long long entries;
};

// Which of a thread's four pages of a chunk are held, as bits.
__device__ __forceinline__ int held_bits(const CompactArgs& a, int chunk) {
  const int p = chunk * kChunk + 4 * threadIdx.x;
  int bits = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) bits |= (p + i < a.num_pages && a.refs[p + i] > 0) << i;
  return bits;
}

// Held pages in all and in front of page n_live, of `before` in front of the chunk. 1024 threads.
__device__ __forceinline__ void compact_sums(const CompactArgs& a, int chunk, int (*part)[16], int* n_live,
                                             int* before, int* low) {
  int all = 0, front = 0;
  for (int i = threadIdx.x; i < a.chunks; i += 1024) {
    all += a.live[i];
    front += i < chunk ? a.live[i] : 0;
  }
  block_scan(all, part[0], n_live);
  block_scan(front, part[1], before);
  *n_live = pages::within(*n_live, a.num_pages);
  const int edge = *n_live / kChunk;  // the chunk that page n_live lies in
  int below = 0;
  for (int i = threadIdx.x; i < edge; i += 1024) below += a.live[i];
  if (edge < a.chunks) {
    const int left = *n_live - edge * kChunk - 4 * (int)threadIdx.x;  // of the thread's pages in front of it
    below += __builtin_popcount(held_bits(a, edge) & ((1 << (left < 0 ? 0 : left > 4 ? 4 : left)) - 1));
  }
  block_scan(below, part[2], low);
}

__device__ __forceinline__ void compact_rank(const CompactArgs& a, int chunk, int (*part)[16], int n_live, int before,
                                             int low) {
  const int most = a.num_pages / 2, bits = held_bits(a, chunk), p0 = chunk * kChunk + 4 * threadIdx.x;
  int total;
  int at = before + block_scan(__builtin_popcount(bits), part[3], &total);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int p = p0 + i;
    if (p >= a.num_pages) break;
    const bool held = bits >> i & 1;
    int rank = -1;
    if (held && p >= n_live) rank = at - low;
    if (!held && p < n_live) rank = p - at;
    a.rank[p] = rank;
    if (rank >= 0 && rank < most) {
      a.moves[(held ? 0 : most) + rank] = p;
      if (held) a.moves[2 * most + rank] = a.refs[p];
    }
    at += held;
  }
}

__device__ __forceinline__ void compact_apply(const CompactArgs& a, int moved, int n_live, long long at,
                                              long long step) {
  const int most = a.num_pages / 2;
  moved = pages::within(moved, most);
  n_live = pages::within(n_live, a.num_pages);
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

__global__ void __launch_bounds__(1024) k_compact_count(const CompactArgs a) {
  __shared__ int part[16];
  int total;
  block_scan(__builtin_popcount(held_bits(a, blockIdx.x)), part, &total);
  if (threadIdx.x == 0) a.live[blockIdx.x] = total;
}

__global__ void __launch_bounds__(1024) k_compact_rank(const CompactArgs a) {
  __shared__ int part[4][16];
  int n_live, before, low;
  compact_sums(a, blockIdx.x, part, &n_live, &before, &low);
  compact_rank(a, blockIdx.x, part, n_live, before, low);
  if (blockIdx.x == 0 && threadIdx.x == 0) {
    a.counts[0] = n_live - low;
    a.counts[1] = n_live;
  }
}

__global__ void __launch_bounds__(256) k_compact_apply(const CompactArgs a) {
  compact_apply(a, a.counts[0], a.counts[1], (long long)blockIdx.x * 256 + threadIdx.x,
                (long long)gridDim.x * 256);
}

// The three of them by one block, for a pool of one chunk.
__global__ void __launch_bounds__(1024) k_compact(const CompactArgs a) {
  __shared__ int part[4][16];
  int n_live, low;
  const int bits = held_bits(a, 0);
  block_scan(__builtin_popcount(bits), part[0], &n_live);
  const int left = n_live - 4 * (int)threadIdx.x;
  block_scan(__builtin_popcount(bits & ((1 << (left < 0 ? 0 : left > 4 ? 4 : left)) - 1)), part[1], &low);
  compact_rank(a, 0, part, n_live, 0, low);
  if (threadIdx.x == 0) {
    a.counts[0] = n_live - low;
    a.counts[1] = n_live;
  }
  __syncthreads();
  compact_apply(a, n_live - low, n_live, threadIdx.x, 1024);
}

// Whether one block does it all: the launches cost more than the other CUs would give. A fork of 8 to 8 sequences
// by tables of 20 pages takes 6.7 us and not 8.8, of 32 to 32 10.6 and 9.9, by 128 pages 11.8 and 10.4 (but two
// launches less, 3 us, on the host), of 64 to 64 by 20 pages 16.4 and 9.8. A compaction of 1000 pages and 1920
// entries 5.1 us and not 8.6, of 4096 and 8192 10.6 and 11.6, of 4096 and 32768 20.4 and 11.6.
bool fork_by_one_block(int n_old, int n_new, int max_pages) {
  return n_old + n_new <= 64 && (n_old + n_new) * max_pages <= 8192;
}
bool compact_by_one_block(int num_pages, long long entries) { return num_pages <= kChunk && entries <= 8192; }

// Whether two arrays of ints share memory.
bool overlap(const int32_t* a, size_t n, const int32_t* b, size_t m) {
  const uintptr_t x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(b);
  return a && b && n && m && x < y + 4 * m && y < x + 4 * n;
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
  size_t all = 0;  // pieces of a pair in all pools
  for (int i = 0; i < n_pools; ++i) {
    if (!pools[i] || page_bytes[i] == 0) return LLMK_ERR_INVALID_VALUE;
    if (page_bytes[i] % 4) return LLMK_ERR_SHAPE;
    if (reinterpret_cast<uintptr_t>(pools[i]) % 4) return LLMK_ERR_ALIGNMENT;
    if (page_bytes[i] > ((size_t)1 << 32)) return LLMK_ERR_UNSUPPORTED;
    all += (page_bytes[i] + kPiece - 1) / kPiece;
  }
  const auto whole = [&](int p) { return aligned16(pools[p]) && page_bytes[p] % 16 == 0; };
  // Many pairs are walked pool by pool, in whose order a compaction's lie in memory: 1024 pairs of 16 KB in 32 pools
  // take 178 us and not 195 in order, 202 and not 214 at random; but 128 pairs in 4 pools 4.9 and not 4.5, 32 pairs of
  // 8 KB in 32 pools 5.5 and not 3.4.
  const bool across = n_copies >= 512;
  // small pages of whole vectors, all of one size, go together
  size_t small = 0;
  for (int p = 0; p < n_pools && !small; ++p)
    if (whole(p) && page_bytes[p] <= 512) small = page_bytes[p];
  // where a launch might not take its blocks, all are counted before the first one
  for (int pass = grid_takes((size_t)n_copies * ((all + 3) / 4), 256) ? 1 : 0; pass < 2; ++pass)
    for (int kind = 0; kind < 2; ++kind)  // whole vectors, then what is not
      for (int i = 0; i < n_pools;) {
        CopyArgs a{};
        a.copies = copies;
        a.count = count;
        a.n_copies = n_copies;
        a.num_pages = num_pages;
        a.across = across;
        int taken = 0;
        const int begin = i;
        for (; i < n_pools && taken < kPools; ++i) taken += whole(i) == (kind == 0);
        if (taken == 0) break;
        const auto is_small = [&](int p) { return kind == 0 && small && page_bytes[p] == small; };
        for (int p = begin; p < i; ++p) {
          if (whole(p) != (kind == 0) || is_small(p)) continue;
          const int n = a.n_pools++;
          a.pool[n] = static_cast<unsigned char*>(pools[p]);
          a.bytes[n] = page_bytes[p];
          a.first[n + 1] = a.first[n] + (int)((page_bytes[p] + kPiece - 1) / kPiece);
        }
        for (int p = begin; p < i; ++p)
          if (whole(p) && is_small(p)) a.pool[a.n_pools + a.n_small++] = static_cast<unsigned char*>(pools[p]);
        a.small = a.n_small ? (int)small : 0;
        size_t pieces = a.first[a.n_pools];
        if (a.n_small) pieces += ceil_div(a.n_small, 64 / (a.small / 16));
        a.slices = (int)((pieces + 3) / 4);
        a.each = a.first[1];
        for (int p = 0; p < a.n_pools; ++p)
          if (a.first[p + 1] - a.first[p] != a.each) a.each = 0;
        const size_t blocks = (size_t)n_copies * a.slices;
        if (!grid_takes(blocks, 256)) return LLMK_ERR_UNSUPPORTED;
        if (pass == 0) continue;
        const int st = launch(kind == 0 ? k_copy_pages<true> : k_copy_pages<false>, dim3((unsigned)blocks),
                              dim3(256), 0, static_cast<hipStream_t>(stream), a);
        if (st != LLMK_OK) return st;
      }
  return LLMK_OK;
}

extern "C" size_t llmk_kv_fork_workspace_ints(int n_old, int n_new, int max_pages, int num_pages) {
  if (n_old < 0 || n_new < 0 || max_pages <= 0 || num_pages <= 0) return 0;
  return 2 + (size_t)n_new * (2 * (size_t)max_pages + 1);
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
  if (n_old > 65535 || n_new > 65535 || max_pages > pages::kMostWanted || num_pages > kMostPages)
    return LLMK_ERR_UNSUPPORTED;
  {  // what is written, and what else there is
    const size_t n = n_new, m = n_old, width = max_pages;
    const int32_t* at[] = {refs,   new_tables, new_lens,     copies,   counts,
                           workspace, block_tables, seq_lens, parents, reserve};
    const size_t size[] = {(size_t)num_pages, n * width, n, 2 * n, 2,
                           llmk_kv_fork_workspace_ints(n_old, n_new, max_pages, num_pages), m * width, m, n, n};
    for (int i = 0; i < 6; ++i)
      for (int j = i + 1; j < 10; ++j)
        if (overlap(at[i], size[i], at[j], size[j])) return LLMK_ERR_INVALID_VALUE;
  }
  if (reinterpret_cast<uintptr_t>(workspace) % 8) return LLMK_ERR_ALIGNMENT;
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
  a.columns = reinterpret_cast<pages::Column*>(workspace + n_new + (n_new & 1));
  a.n_old = n_old;
  a.n_new = n_new;
  a.max_pages = max_pages;
  a.page_size = page_size;
  a.num_pages = num_pages;
  if (fork_by_one_block(n_old, n_new, max_pages)) return launch(k_fork, dim3(1), dim3(1024), 0, s, a);
  // Entries a lane has on their way, 1, 4 and 16: 32 to 32 sequences by tables of 20 pages take 9.9, 10.4 and 13.0 us,
  // 256 by 130 14.0, 13.3 and 15.7, 32 by 257 13.5, 12.4 and 13.8, by 1024 25.9, 21.9 and 18.5.
  const int entries = max_pages <= 128 ? 1 : max_pages <= 512 ? 4 : 16;
  int st = LLMK_OK;
  if (n_new > 0)
    st = launch(entries == 1 ? k_fork_rows<1> : entries == 4 ? k_fork_rows<4> : k_fork_rows<16>,
                dim3(ceil_div(n_new, 4)), dim3(256), 0, s, a);
  if (st == LLMK_OK && n_old > 0)
    st = launch(entries == 1 ? k_fork_refs<1> : entries == 4 ? k_fork_refs<4> : k_fork_refs<16>,
                dim3(ceil_div(n_old, 4)), dim3(256), 0, s, a);
  if (st == LLMK_OK) st = launch(k_fork_find, dim3(1), dim3(1024), 0, s, a);
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
  {
    const size_t pages = num_pages, entries = (size_t)n_seqs * max_pages;
    const int32_t* at[] = {new_tables, new_refs, copies, counts, workspace, block_tables, refs};
    const size_t size[] = {entries, pages, 2 * (pages / 2), 2, llmk_kv_compact_workspace_ints(num_pages),
                           entries, pages};
    for (int i = 0; i < 5; ++i)
      for (int j = i + 1; j < 7; ++j) {
        const bool same = at[i] == at[j] && ((i == 0 && j == 5) || (i == 1 && j == 6));
        if (!same && overlap(at[i], size[i], at[j], size[j])) return LLMK_ERR_INVALID_VALUE;
      }
  }
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
  if (compact_by_one_block(num_pages, a.entries)) return launch(k_compact, dim3(1), dim3(1024), 0, s, a);
  int st = launch(k_compact_count, dim3(a.chunks), dim3(1024), 0, s, a);
  if (st == LLMK_OK) st = launch(k_compact_rank, dim3(a.chunks), dim3(1024), 0, s, a);
  if (st != LLMK_OK) return st;
  const long long most = a.entries > num_pages ? a.entries : num_pages;
  const long long blocks = (most + 255) / 256;
  return launch(k_compact_apply, dim3((unsigned)(blocks < 2048 ? blocks : 2048)), dim3(256), 0, s, a);
}
