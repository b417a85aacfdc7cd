"""What the join of llmk_kv8_attention makes of its notes in the workspace, whatever they hold: addresses
inside the workspace and the output. The check is host code; the join's indices are restated here, on
the CPU."""
import os
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                    "cuda-llm-engine_amd", "csrc")

SOURCE = r"""
#include <cstdio>
#include <random>

#include "kv8_shared.hpp"
using llmk::kv8::Shared;
using llmk::kv8::is_unit;
using llmk::kv8::row_of;

int main() {
  std::mt19937 rng(7);
  auto any = [&](long long lo, long long hi) {
    return (int)std::uniform_int_distribution<long long>(lo, hi)(rng);
  };
  // a number that is small, next to one of the call's own, or anything
  auto odd = [&](int a, int b) {
    switch (any(0, 5)) {
      case 0: return any(-3, 3);
      case 1: return any(a - 2LL, a + 2LL) ;
      case 2: return any(b - 2LL, b + 2LL);
      case 3: return any(0, a > 1 ? a : 1);
      case 4: return any(0, 3) == 0 ? (int)0x7FC00000 : (int)0x80000000;
      default: return any(-2147483648LL, 2147483647LL);
    }
  };
  long long kept = 0, rows = 0;
  for (int turn = 0; turn < 3000000; ++turn) {
    const int most = 16 << any(0, 4), heads = any(1, 12), workers = any(heads, 2048);
    const int teams = workers / heads, group = any(1, 40), n_rows = any(1, 3000);
    const int team = any(0, teams - 1);
    Shared o = {odd(teams, team), odd(teams, team), odd(n_rows * group, most), odd(most, n_rows),
                odd(n_rows, n_rows - 1), odd(most, 0), {0, 0}};
    if (!is_unit(o, team, teams, most)) continue;
    ++kept;
    const long long first = ((long long)o.first * heads * 2 + 1) * most;
    const long long last = (2LL * ((long long)o.last * heads + heads - 1) + 1) * most + o.columns - 1;
    const long long slice = team - o.first, n = (long long)o.last - o.first + 1;
    bool good = first >= 0 && last < 2LL * workers * most && slice >= 0 && slice < n && n <= workers;
    for (int c : {0, (o.columns - 1) / 2, o.columns - 1}) {
      const long long col = (long long)o.column + c, row = o.row0 + col / group;
      const bool inside = o.row0 >= 0 && row < n_rows;
      good = good && col % group >= 0 && row_of(o, c, n_rows, group) == (inside ? row : -1);
      rows += inside;
    }
    if (!good) {
      std::printf("%d %d %d %d %d of %d teams, %d columns, %d rows\n", o.first, o.last, o.column,
                  o.columns, o.row0, teams, most, n_rows);
      return 1;
    }
  }
  if (kept < 1000 || rows < 1000) return 2;
  // notes as workers make them
  const Shared none = {0, -1, 0, 0, 0, 0, {0, 0}};
  const Shared all = {0, 127, 992, 32, 3, 0, {0, 0}};  // the last columns of 256 rows from row 3 on
  if (is_unit(none, 0, 128, 32)) return 3;
  for (int team = 0; team < 128; ++team)
    if (!is_unit(all, team, 128, 32)) return 4;
  if (is_unit(all, 0, 127, 32) || is_unit(all, 0, 128, 16)) return 5;
  for (int c = 0; c < 32; ++c)
    if (row_of(all, c, 259, 4) != 251 + c / 4 || row_of(all, c, 251 + c / 4, 4) != -1) return 6;
  return 0;
}
"""


@pytest.fixture(scope="module")
def program(tmp_path_factory):
    at = tmp_path_factory.mktemp("shared")
    (at / "shared.cpp").write_text(SOURCE)
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Werror", "-I", CSRC,
                    str(at / "shared.cpp"), "-o", str(at / "shared")], check=True)
    return str(at / "shared")


def test_notes_of_any_content_stay_inside(program):
    r = subprocess.run([program], capture_output=True, text=True)
    assert r.returncode == 0, (r.returncode, r.stdout)
