"""Kernel attributes are set on every device that a process uses: the helper of the paged
attention's launches against a stand-in for the two runtime calls it makes, and both
launches through it."""
import os
import re
import shutil
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(__file__), "..", "thunderllamax_b200", "csrc")
INCLUDE = "/usr/local/cuda/include"
PROGRAM = r"""
#include "kernel_setup.h"
#include <cstdio>
static int device = 0, calls = 0;
static bool fails = false;
extern "C" cudaError_t cudaGetDevice(int* d) { *d = device; return cudaSuccess; }
extern "C" cudaError_t cudaFuncSetAttribute(const void*, cudaFuncAttribute, int) {
  ++calls;
  return fails ? cudaErrorInvalidValue : cudaSuccess;
}
#define EXPECT(c) do { if (!(c)) { std::printf("line %d: %s\n", __LINE__, #c); return 1; } } while (0)
int main() {
  std::atomic<uint64_t> done{0}, other{0};
  EXPECT(tlx::setup_kernel(nullptr, 1000, done) && calls == 2);
  EXPECT(tlx::setup_kernel(nullptr, 1000, done) && calls == 2);    // once on a device
  device = 1;
  EXPECT(tlx::setup_kernel(nullptr, 1000, done) && calls == 4);    // and on the next one
  EXPECT(tlx::setup_kernel(nullptr, 1000, done) && calls == 4);
  EXPECT(tlx::setup_kernel(nullptr, 1000, other) && calls == 6);   // another kernel
  device = 2;
  fails = true;
  EXPECT(!tlx::setup_kernel(nullptr, 1000, done) && calls == 7);   // a refusal is not taken for done
  fails = false;
  EXPECT(tlx::setup_kernel(nullptr, 1000, done) && calls == 9);
  device = 70;
  EXPECT(tlx::setup_kernel(nullptr, 1000, done) && tlx::setup_kernel(nullptr, 1000, done) && calls == 13);
  return 0;
}
"""


@pytest.mark.skipif(not shutil.which("g++") or not os.path.exists(INCLUDE), reason="needs g++ and the CUDA headers")
def test_attributes_are_set_on_each_device(tmp_path):
    src = tmp_path / "setup.cpp"
    src.write_text(PROGRAM)
    exe = str(tmp_path / "setup")
    subprocess.run(["g++", "-std=c++17", f"-I{CSRC}", f"-I{INCLUDE}", str(src), "-o", exe], check=True)
    got = subprocess.run([exe], capture_output=True, text=True)
    assert got.returncode == 0, got.stdout


@pytest.mark.parametrize("name", ["paged_rows.cu", "paged_tiles.cu"])
def test_launches_go_through_it(name):
    src = open(os.path.join(CSRC, name)).read()
    assert "setup_kernel(" in src and "cudaFuncSetAttribute" not in src
    assert not re.search(r"static bool \w+ = false", src)
