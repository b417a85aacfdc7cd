"""What the steps of llmk_kv_fork count and leave one another (csrc/fork_notes.hpp): host code, compiled for the
CPU; the kernels' uses of it are restated here."""
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
