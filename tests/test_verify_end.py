"""What llmk_verify_drafts makes of the ends of sequences in its workspace, whatever they hold: rows of the
call. Host code, on the CPU; the kernels' uses of an end are restated here."""
import os
import subprocess

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                    "cuda-llm-engine_amd", "csrc")

SOURCE = r"""
#include <cstdio>
#include <random>

#include "verify_end.hpp"
using llmk::verify::End;
using llmk::verify::checked;

int main() {
  std::mt19937 rng(8);
  auto any = [&](long long lo, long long hi) {
    return (int)std::uniform_int_distribution<long long>(lo, hi)(rng);
  };
  auto odd = [&](int a) {
    switch (any(0, 3)) {
      case 0: return any(a - 2LL, a + 2LL);
      case 1: return any(-2, a);
      case 2: return any(0, 1) == 0 ? (int)0x7FC00000 : (int)0x80000000;
      default: return any(-2147483648LL, 2147483647LL);
    }
  };
  long long drawn = 0;
  for (int turn = 0; turn < 3000000; ++turn) {
    const bool starts = any(0, 1) == 0;
    const int n_rows = any(1, 500), s = any(0, n_rows - 1);
    const End was = {odd(s), odd(n_rows), odd(s), any(0, 1), any(0, 1), odd(s), 0, 0, {0, 0, 0}};
    const End z = checked(was, s, starts, n_rows);
    bool good = true;
    if (z.end > z.first) {  // tokens of all its rows, drafts in front of its last one
      good = z.first >= 0 && z.end <= n_rows && z.row >= z.first && z.row < z.end;
      if (!starts) good = good && z.first == s && z.end == s + 1 && z.last;
      good = good && z.last == (z.row == z.end - 1) && z.row == was.row;
      ++drawn;
    }
    // a row to draw from
    if (z.row >= z.first) good = good && z.end > z.first;
    if (!good) {
      std::printf("%d %d %d, sequence %d of %d rows\n", was.first, was.end, was.row, s, n_rows);
      return 1;
    }
  }
  if (drawn < 1000) return 2;
  // ends as they are found stay as they are
  for (int first = 0; first < 5; ++first)
    for (int end = first; end < 8; ++end)
      for (int row = end > first ? first : end - 1; row < end || row == end - 1; ++row) {
        const End z = checked({first, end, row, row == end - 1, 0, 3, 0, 0, {0, 0, 0}}, 2, true, 7);
        if (z.first != first || z.end != end || z.row != row || z.last != (row == end - 1)) return 3;
        if (row == end - 1) break;
      }
  return 0;
}
"""


def test_ends_of_any_content_are_rows_of_the_call(tmp_path):
    (tmp_path / "end.cpp").write_text(SOURCE)
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Werror", "-I", CSRC,
                    str(tmp_path / "end.cpp"), "-o", str(tmp_path / "end")], check=True)
    r = subprocess.run([str(tmp_path / "end")], capture_output=True, text=True)
    assert r.returncode == 0, (r.returncode, r.stdout)
