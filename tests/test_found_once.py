"""Host-side facts that are found once (``csrc/found_once.h``): only a search that succeeded is kept."""

import os
import shutil
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "csrc")

PROGRAM = """
#include "found_once.h"
int main() {
  dfl_host::FoundOnce<int> fact;
  int searches = 0, value = -1;
  auto failing = [&](int* v) { ++searches; *v = 5; return 719; };
  auto found = [&](int* v) { ++searches; *v = 7; return 0; };
  if (fact.get(&value, failing) != 719 || value != -1) return 1;
  if (fact.get(&value, found) != 0 || value != 7 || searches != 2) return 2;
  if (fact.get(&value, failing) != 0 || value != 7 || searches != 2) return 3;
  return 0;
}
"""


def test_a_failed_search_is_tried_again(tmp_path):
    cxx = shutil.which("g++")
    if cxx is None:
        pytest.skip("no C++ compiler")
    src = tmp_path / "main.cpp"
    src.write_text(PROGRAM)
    subprocess.run([cxx, "-std=c++17", "-I", CSRC, str(src), "-o", str(tmp_path / "main"), "-pthread"], check=True)
    assert subprocess.run([str(tmp_path / "main")]).returncode == 0


def test_occupancy_of_the_few_query_kernel_is_found_that_way():
    """(call_once with the error stored beside it refused every later call after one transient failure.)"""
    with open(os.path.join(CSRC, "cross_decode.cu")) as f:
        source = f.read()
    assert "FoundOnce" in source and "call_once" not in source
