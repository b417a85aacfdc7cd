"""Whether rows of pieces share memory (csrc/overlap.hpp, host arithmetic), against sets of addresses. On the CPU."""
import os
import random
import subprocess

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "cuda-llm-engine_amd", "csrc")
SOURCE = r"""
#include <stdio.h>
#include "overlap.hpp"
using namespace llmk;
int main() {
  long long v[12];
  for (;;) {
    for (auto& x : v)
      if (scanf("%lld", &x) != 1) return 0;
    const Rows a{(uintptr_t)v[0], v[1], v[2], v[3], v[4], v[5]}, b{(uintptr_t)v[6], v[7], v[8], v[9], v[10], v[11]};
    printf("%d %d\n", overlap(a, b), overlap(b, a));
  }
}
"""


def elements(at, n, ld, pieces, apart, width):
    return {at // 2 + r * ld + p * apart + e for r in range(n) for p in range(pieces) for e in range(width)}


def test_against_sets(tmp_path):
    (tmp_path / "o.cpp").write_text(SOURCE)
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Werror", "-I", CSRC, str(tmp_path / "o.cpp"), "-o",
                    str(tmp_path / "o")], check=True)
    rng, cases = random.Random(2), []
    for _ in range(40000):
        both = []
        ld_of_both = rng.randint(1, 30)
        for _ in range(2):
            pieces, width = rng.randint(1, 4), rng.randint(1, 5)
            apart = width + rng.randint(0, 6)
            row = (pieces - 1) * apart + width
            ld = max(row, ld_of_both) + (rng.randint(0, 3) if rng.random() < 0.4 else 0)
            both.append([2 * rng.randint(100, 100 + rng.choice([10, 150])), rng.randint(1, 5), ld, pieces, apart, width])
        if rng.random() < 0.5:  # columns of one matrix
            both[0][2] = both[1][2] = max(both[0][2], both[1][2])
        elif rng.random() < 0.3:  # a contiguous array
            both[1] = [both[1][0], 1, 0, 1, 1, 1]
            both[1][4] = both[1][5] = rng.randint(1, 40)
        cases.append(both[0] + both[1])
    cases.append([0, 1, 5, 1, 5, 5, 0, 1, 5, 1, 5, 5])  # arrays that are not there
    cases.append([64, 0, 5, 1, 5, 5, 64, 1, 5, 1, 5, 5])
    out = subprocess.run([str(tmp_path / "o")], input="\n".join(" ".join(map(str, c)) for c in cases),
                         capture_output=True, text=True, check=True).stdout.split()
    hits = 0
    for c, ab, ba in zip(cases, out[::2], out[1::2], strict=True):
        want = bool(c[0]) and bool(elements(*c[:6]) & elements(*c[6:]))
        hits += want
        assert (int(ab), int(ba)) == (want, want), c
    assert 5000 < hits < 35000
