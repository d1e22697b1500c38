"""Two host threads that launch one kernel for the first time with different amounts of shared memory: what is noted as granted is
never more than what the kernel's attribute is left at.  The CUDA calls are fakes that meet in the order that used to lose one."""
import os
import subprocess

from tests._util import ROOT

PROGRAM = r"""
#include <atomic>
#include <chrono>
#include <cstdio>
#include <thread>

#include "blkq4_tma.cuh"

static std::atomic<int> attribute{0};
static std::atomic<bool> large_set{false}, small_done{false};
static bool meet = true;

static void await(std::atomic<bool>& flag) {  // or half a second, where the other one is kept out
  for (int i = 0; i < 500 && !flag.load(); ++i) std::this_thread::sleep_for(std::chrono::milliseconds(1));
}
extern "C" cudaError_t cudaGetDevice(int* dev) { *dev = 0; return cudaSuccess; }
extern "C" cudaError_t cudaFuncSetAttribute(const void*, cudaFuncAttribute, int bytes) {
  if (meet && bytes == 100) await(large_set);
  attribute = bytes;
  if (meet && bytes == 200) { large_set = true; await(small_done); }
  return cudaSuccess;
}

int main() {
  static std::atomic<int> granted[64];
  const void* kernel = nullptr;
  std::thread small([&] { blkq4::ensure_dynamic_smem(kernel, 100, granted); small_done = true; });
  std::thread large([&] { blkq4::ensure_dynamic_smem(kernel, 200, granted); });
  small.join();
  large.join();
  meet = false;
  for (int want : {180, 50, 250, 220}) {
    if (blkq4::ensure_dynamic_smem(kernel, want, granted) != cudaSuccess || attribute.load() < want) {
      std::printf("%d bytes wanted, %d granted, the attribute is %d\n", want, granted[0].load(), attribute.load());
      return 1;
    }
  }
  return 0;
}
"""


def test_the_attribute_is_only_raised(tmp_path):
    from gemmlib_b200 import build

    cuda = os.path.dirname(os.path.dirname(os.path.realpath(build._nvcc())))
    src, exe = tmp_path / "grant.cpp", tmp_path / "grant"
    src.write_text(PROGRAM)
    subprocess.run(["g++", "-std=c++17", "-O1", "-pthread", "-I" + os.path.join(cuda, "include"),
                    "-I" + os.path.join(ROOT, "gemmlib_b200", "csrc"), str(src), "-o", str(exe)], check=True, timeout=120)
    r = subprocess.run([str(exe)], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0, r.stdout + r.stderr
