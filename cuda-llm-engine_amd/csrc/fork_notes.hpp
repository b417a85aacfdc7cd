// What the steps of llmk_kv_fork count and leave one another. No device code: a program on the host may
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

}  // namespace pages
}  // namespace llmk
