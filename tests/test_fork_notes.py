"""What the steps of llmk_kv_fork and llmk_kv_compact count and leave one another (csrc/fork_notes.hpp): host code,
compiled for the CPU; the kernels' uses of it are restated here."""
import os
import random
import subprocess

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                    "cuda-llm-engine_amd", "csrc")

SUMS = r"""
#include <cstdio>
#include "fork_notes.hpp"
int main() {  // in: children and the pages that each wants; out: pages wanted in front of each, and by all
  int n;
  long long wanted = 0;
  if (std::scanf("%d", &n) != 1) return 1;
  for (int c0 = 0; c0 < n; c0 += 1024) {
    int mine[1024] = {}, part[16];
    for (int c = c0; c < n && c < c0 + 1024; ++c)
      if (std::scanf("%d", &mine[c - c0]) != 1) return 1;
    for (int w = 0; w < 16; ++w) {
      part[w] = 0;
      for (int i = 0; i < 64; ++i)
        if (__builtin_add_overflow(part[w], mine[64 * w + i], &part[w])) return 2;
    }
    long long total = 0;
    for (int w = 0; w < 16; ++w) {
      const auto s = llmk::pages::sums_of<long long>(part, 16, w);
      long long at = wanted + s.before;
      total = s.all;
      for (int i = 0; i < 64 && c0 + 64 * w + i < n; at += mine[64 * w + i++]) std::printf("%lld\n", at);
    }
    wanted += total;
  }
  std::printf("%lld\n", wanted);
}
"""

NOTES = r"""
#include <cstdio>
#include <random>
#include "fork_notes.hpp"
using namespace llmk::pages;
int main() {  // whatever the workspace holds, what is read and written is the call's
  std::mt19937 rng(5);
  auto any = [&](long long lo, long long hi) { return (int)std::uniform_int_distribution<long long>(lo, hi)(rng); };
  auto odd = [&](int a) {
    switch (any(0, 3)) {
      case 0: return any(a - 2LL, a + 2LL);
      case 1: return any(-2, a);
      case 2: return any(0, 1) == 0 ? (int)0x80000000 : 0x7FFFFFFF;
      default: return any(-2147483648LL, 2147483647LL);
    }
  };
  for (int turn = 0; turn < 2000000; ++turn) {
    const int max_pages = any(0, 1) ? any(1, 9) : kMostWanted, num_pages = any(1, 30);
    const int noted = odd(max_pages), wanted = wanted_of(noted, max_pages);
    if (wanted < 0 || wanted > max_pages) return 1;
    const Column c = checked({odd(max_pages), odd(num_pages)}, max_pages, num_pages);
    if (c.at < -1 || c.at >= max_pages || c.from < -1 || c.from >= num_pages) return 2;
    if (c.at < 0 && c.from >= 0) return 3;
    const int at = place_of(any(0, num_pages - 1), odd(num_pages), max_pages);
    if (at < 0 || at >= max_pages) return 4;
  }
  // what the steps themselves note stays as it is
  for (int n : {0, 1, 5, kMostWanted})
    for (int beside : {0, kCopiesShared})
      if (wanted_of(n + beside, kMostWanted) != n) return 5;
  for (int j = 0; j < 6; ++j)
    for (int page = -1; page < 9; ++page) {
      const Column c = checked({j, page}, 6, 9);
      if (c.at != j || c.from != page) return 6;
    }
  for (int begin = 0; begin < 5; ++begin)
    for (int k = begin; k < begin + 6; ++k)
      if (place_of(k, begin, 6) != k - begin) return 7;
  return 0;
}
"""

COMPACT = r"""
#include <cstdio>
#include <random>
#include "fork_notes.hpp"
using namespace llmk::pages;
int main() {  // the places that the steps read and write, whatever the workspace and the counts hold
  std::mt19937 rng(6);
  auto any = [&](long long lo, long long hi) { return (int)std::uniform_int_distribution<long long>(lo, hi)(rng); };
  auto odd = [&](int a) {
    switch (any(0, 3)) {
      case 0: return any(a - 2LL, a + 2LL);
      case 1: return any(-2, a);
      case 2: return any(0, 1) == 0 ? (int)0x80000000 : 0x7FFFFFFF;
      default: return any(-2147483648LL, 2147483647LL);
    }
  };
  for (int turn = 0; turn < 2000000; ++turn) {
    const int num_pages = any(0, 1) ? any(1, 20000) : any(1, 1 << 24), most = num_pages / 2;
    const int chunks = (num_pages + 4095) / 4096;
    const int edge = within(odd(num_pages), num_pages) / 4096;
    if (edge < 0 || edge > chunks) return 1;  // sums of chunks below it; its own counts if it is below `chunks`
    const int moved = within(odd(most), most), n_live = within(odd(num_pages), num_pages);
    const int p = odd(num_pages), rank = odd(most);
    if (p >= n_live && p < num_pages && p < 0) return 2;  // a table's entry becomes an address
    if ((unsigned)rank < (unsigned)moved && (rank < 0 || rank >= most)) return 3;
  }
  for (int n = 0; n <= 9; ++n)
    if (within(n, 9) != n) return 4;
  return 0;
}
"""


def program(tmp_path, source):
    (tmp_path / "main.cpp").write_text(source)
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Werror", "-I", CSRC, str(tmp_path / "main.cpp"), "-o",
                    str(tmp_path / "main")], check=True)
    return str(tmp_path / "main")


def test_sums_past_32_bits(tmp_path):
    """Each child may want 2^24 pages, a block's children 2^34."""
    run = program(tmp_path, SUMS)
    rng = random.Random(3)
    for wants in ([2 ** 21] * 1024, [2 ** 22 + 1024] * 1024, [2 ** 24] * 3000, [5], [0] * 70,
                  [rng.choice([0, 1, 7, 2 ** 23, 2 ** 24]) for _ in range(2500)]):
        out = subprocess.run([run], input=" ".join(map(str, [len(wants), *wants])), capture_output=True, text=True,
                             check=True).stdout
        assert [int(x) for x in out.split()] == [sum(wants[:c]) for c in range(len(wants) + 1)]


def test_notes_of_any_content_are_places_of_the_call(tmp_path):
    r = subprocess.run([program(tmp_path, NOTES)])
    assert r.returncode == 0


def test_counts_of_any_content_are_places_of_the_call(tmp_path):
    r = subprocess.run([program(tmp_path, COMPACT)])
    assert r.returncode == 0
