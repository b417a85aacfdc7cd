"""The C++ names of adapters, rotary layouts and shared pages: what they take, and that they refuse as the
others do (the message, exit code 1). Refusals come before any launch: no GPU is needed."""
import os
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
PACKAGE = os.path.join(ROOT, "cuda-llm-engine_amd")

SOURCE = r"""
#include "llmk.hpp"
int main(int argc, char** argv) {
  const __half* in = nullptr;
  __half* out = nullptr;
  float* f = nullptr;
  int* ints = nullptr;
  const int ends[] = {8, 24};
  void* pools[] = {nullptr};
  const size_t bytes[] = {64};
  const bool bad = argc > 2;
  switch (argv[1][0]) {
    case 'l': lora_add(in, 64, in, in, ints, f, ints, ints, out, 24, ends, bad ? 9 : 2, f, 0, 0, 1, 16, 64); break;
    case 'r': rotary_apply(out, 64, out, 64, ints, f, ints, f, 0, 1, 1, 64, bad ? 66 : 64, 1, LLMK_ROTARY_PAIRS); break;
    case 's': qkv_rotary_scatter(in, 192, out, out, out, ints, ints, f, ints, f, 0, 1, 16, 1, 1, 64, bad ? 24 : 64, 1, LLMK_ROTARY_HALVES); break;
    case 'i': return compute_rotary_inv_freq(LLMK_ROTARY_YARN, bad ? 63 : 64, 1e4, 4.0, 4096.0, 32.0, 1.0, f).size() == 32 ? 0 : 2;
    case 'c': kv_copy_pages(pools, bytes, 1, ints, nullptr, 0, bad ? 0 : 8); break;
    case 'f': kv_fork(ints, ints, ints, nullptr, ints, ints, ints, ints, ints, ints, bad ? -1 : 65536, 1, 1, 16, 8); break;
    case 'k': kv_compact(ints, ints, ints, ints, ints, ints, ints, 1, 1, bad ? 0 : 8); break;
    default:
      return lora_add_workspace_floats(1, 1, 1, 8, 8, 1) > 0 && kv_fork_workspace_ints(1, 1, 1, 1) > 0 &&
                     kv_compact_workspace_ints(8) > 0 && kv_compact_workspace_ints(0) == 0
                 ? 0
                 : 2;
  }
  return 0;
}
"""


@pytest.fixture(scope="module")
def program(tmp_path_factory, llmk):
    at = tmp_path_factory.mktemp("shims")
    (at / "shims.cpp").write_text(SOURCE)
    subprocess.run(["g++", "-std=c++17", "-Wall", "-Werror", "-D__HIP_PLATFORM_AMD__", "-isystem",
                    "/opt/rocm/include", "-I", os.path.join(ROOT, "include"), str(at / "shims.cpp"),
                    "-o", str(at / "shims"), "-L", PACKAGE, "-lllmk", f"-Wl,-rpath,{PACKAGE}",
                    "-L/opt/rocm/lib", "-lamdhip64", "-Wl,-rpath,/opt/rocm/lib"], check=True)
    return str(at / "shims")


@pytest.mark.parametrize("call,name", [("l", "lora_add"), ("r", "rotary_apply"), ("s", "qkv_rotary_scatter"),
                                       ("i", "compute_rotary_inv_freq"), ("c", "kv_copy_pages")])
def test_a_call_of_nothing_and_a_refused_one(program, call, name):
    assert subprocess.run([program, call]).returncode == 0
    bad = subprocess.run([program, call, "bad"], capture_output=True, text=True)
    assert bad.returncode == 1 and bad.stderr.startswith(name + ":")


@pytest.mark.parametrize("call,name", [("f", "kv_fork"), ("k", "kv_compact")])
def test_refused_ones(program, call, name):
    for args in ([call], [call, "bad"]):  # null arrays, and a size below 1
        bad = subprocess.run([program, *args], capture_output=True, text=True)
        assert bad.returncode == 1 and bad.stderr.startswith(name + ":")


def test_workspace_sizes(program):
    assert subprocess.run([program, "w"]).returncode == 0
