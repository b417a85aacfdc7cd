// What the steps of llmk_kv_fork and llmk_kv_compact count and leave one another. No device code: a program on the host may
// include it.
#pragma once

namespace llmk {
namespace pages {

constexpr int kMostWanted = 1 << 24;  // pages that a child may want: no table is wider

// Sums over a block's waves: in front of one of them, and over all. Wanted pages need 64 bits for T: a wave's 64
// children end below 2^31, a block's 1024 do not.
template <typename T>
struct Sums {
  T before, all;
};
template <typename T>
constexpr Sums<T> sums_of(const int* part, int waves, int wave) {
  Sums<T> s{0, 0};
  for (int w = 0; w < waves; ++w) {
    s.before += w < wave ? part[w] : 0;
    s.all += part[w];
  }
  return s;
}
static_assert(64LL * kMostWanted < 1LL << 31, "a wave's sum in 32 bits");

// In the workspace: how many pages a child wants, and beside it, for a first child that copies a page that others held
// (who may all let go), kCopiesShared; and a column for each wanted page. All become addresses, and the workspace is the
// caller's memory: where another stream's call or a temporary overwrites it between the launches, tables are wrong,
// but nothing that is not the call's is read or written.
constexpr int kCopiesShared = 1 << 30;
constexpr int wanted_of(int noted, int max_pages) {
  const int n = noted & (kCopiesShared - 1);
  return n < max_pages ? n : max_pages;
}

struct alignas(8) Column {
  int at;    // where in the child's row; -1: nowhere
  int from;  // the page that is to be copied; -1: none
};
constexpr Column checked(Column c, int max_pages, int num_pages) {
  if (c.at < 0 || c.at >= max_pages) c.at = c.from = -1;
  if (c.from < 0 || c.from >= num_pages) c.from = -1;
  return c;
}

// The place of the k-th wanted page of all among a child's, whose first one is the begin-th: one of its row's columns.
constexpr int place_of(int k, int begin, int max_pages) {
  const long long at = (long long)k - begin;
  return at < 0 ? 0 : at < max_pages ? (int)at : max_pages - 1;
}

// The same for llmk_kv_compact: its counts are added up from the workspace and pass through `counts`, ranks are
// compared with them where they are used.
constexpr int within(int n, int most) { return n < 0 ? 0 : n < most ? n : most; }

}  // namespace pages
}  // namespace llmk
