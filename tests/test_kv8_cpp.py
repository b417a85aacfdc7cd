"""The C++ names of the 8-bit cache's operators: what they take, and that they refuse as the others do
(the message, exit code 1). Refusals come before any launch: no GPU is needed."""
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
  uint8_t* pool = nullptr;
  float *scale = nullptr, *ws = nullptr;
  int* ints = nullptr;
  const int page = argc > 2 ? 8 : 16;  // 8: refused
  switch (argv[1][0]) {
    case 'a': kv8_append(in, 384, out, pool, scale, pool, scale, ints, nullptr, ints, scale, 0, 0, 1, page, 4, 1, 64); break;
    case 'g': kv8_gather(pool, scale, pool, scale, ints, nullptr, ints, out, out, 0, 0, 1, page, 1, 64); break;
    case 't': kv8_attention(in, pool, scale, pool, scale, ints, nullptr, ints, out, ws, 0, 0, 1, 1, page, 4, 1, 64); break;
    case 'v': verify_drafts(in, in, ints, ints, scale, scale, scale, ints, ints, ws, 0, 0, page == 8 ? 0 : 100); break;
    default:
      return kv8_attention_workspace_floats(64) > 0 && kv8_attention_workspace_floats(65) == 0 &&
                     verify_drafts_workspace_floats(5, 1, 100) > 0
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


@pytest.mark.parametrize("call,name", [("a", "kv8_append"), ("g", "kv8_gather"),
                                       ("t", "kv8_attention"), ("v", "verify_drafts")])
def test_a_call_of_nothing_and_a_refused_one(program, call, name):
    assert subprocess.run([program, call]).returncode == 0
    bad = subprocess.run([program, call, "bad"], capture_output=True, text=True)
    assert bad.returncode == 1 and bad.stderr.startswith(name + ":")


def test_workspace_sizes(program):
    assert subprocess.run([program, "w"]).returncode == 0
