"""Kernel attributes belong to the device that is current when they are set: a second GPU in one process needs them too."""

import pathlib
import re
import shutil
import subprocess

import pytest

CSRC = pathlib.Path(__file__).resolve().parent.parent / "csrc"
PROGRAM = r"""
#include "once.h"
#include <cstdio>
#include <stdexcept>
int main() {
  std::atomic<uint64_t> done{0};
  int ran[80] = {};
  auto on = [&](int d) { qw::once_per_device(done, d, [&] { ++ran[d]; }); };
  for (int i = 0; i < 3; ++i) { on(0); on(1); on(63); on(70); }
  try { qw::once_per_device(done, 2, [] { throw std::runtime_error("no"); }); } catch (const std::runtime_error&) {}
  on(2);
  std::printf("%d %d %d %d %d", ran[0], ran[1], ran[2], ran[63], ran[70]);
}
"""


@pytest.mark.skipif(shutil.which("g++") is None, reason="needs a C++ compiler")
def test_settings_are_made_once_on_each_device(tmp_path):
    (tmp_path / "once.cpp").write_text(PROGRAM)
    subprocess.run(["g++", "-std=c++17", "-I", str(CSRC), "-o", str(tmp_path / "once"), str(tmp_path / "once.cpp")], check=True)
    out = subprocess.run([str(tmp_path / "once")], check=True, capture_output=True, text=True).stdout
    assert out.split() == ["1", "1", "1", "1", "3"]


@pytest.mark.parametrize("name", ["kv_cache.cu", "cached_attention.cu", "cached_attention_tc.cu"])
def test_the_cache_kernels_set_their_attributes_per_device(name):
    source = (CSRC / name).read_text()
    for call in re.finditer(r"cudaFuncSetAttribute", source):
        assert "once_per_device" in source[max(0, call.start() - 400):call.start()], f"{name}: attributes set once per process"
