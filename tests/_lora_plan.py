"""How calls of lora_add are cut into launches (csrc/lora_plan.hpp, host arithmetic), compiled for the CPU."""
import os
import subprocess

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "cuda-llm-engine_amd", "csrc")

SOURCE = r"""
#include <stdio.h>
#include "lora_plan.hpp"
using namespace llmk::lora;
int main() {
  int rows, seqs, adapters, rank, in, parts, ends[kParts];
  while (scanf("%d %d %d %d %d %d", &rows, &seqs, &adapters, &rank, &in, &parts) == 6) {
    for (int p = 0; p < parts; ++p)
      if (scanf("%d", &ends[p]) != 1) return 1;
    const Shape s = shape_of(rows, seqs, adapters, in, parts * ((rank + 15) / 16));
    const Tiles t = tiles_of(rows, seqs, adapters, s.windows, s.groups);
    const Launches l = launches_of(s, rows, seqs, adapters, rank, in, ends, parts);
    printf("%d %d %d %d %d %d %d %d %d %d %d %d %d %d %zu %zu\n", s.groups, s.windows, s.slots, s.splits, s.at_once,
           s.turns, t.likely, t.many, l.one, l.tiles, l.together, l.blocks, l.per_block, l.steps, l.grid, l.grid2);
  }
}
"""
NAMES = ("groups", "windows", "slots", "splits", "at_once", "turns", "likely", "many", "one", "tiles", "together",
         "blocks", "per_block", "steps", "grid", "grid2")


def plans(directory, calls):
    """What becomes of (n_rows, n_seqs, n_adapters, max_rank, in_features, part_ends), a dict each."""
    (directory / "plan.cpp").write_text(SOURCE)
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Werror", "-ftrapv", "-I", CSRC,
                    str(directory / "plan.cpp"), "-o",
                    str(directory / "plan")], check=True)
    text = "\n".join(" ".join(map(str, [*c[:5], len(c[5]), *c[5]])) for c in calls)
    out = subprocess.run([str(directory / "plan")], input=text, capture_output=True, text=True, check=True).stdout
    return [dict(zip(NAMES, map(int, line.split()), strict=True)) for line in out.splitlines()]
