"""A kernel's shared-memory limit under host threads, with the runtime's calls replaced."""
import os
import subprocess

from conftest import PKG

SRC = r"""
#include <cuda_runtime.h>
#include <chrono>
#include <cstdio>
#include <thread>
static std::atomic<int>* limit;
static void rest(int ms) { std::this_thread::sleep_for(std::chrono::milliseconds(ms)); }
static cudaError_t current(int* dev) { *dev = 0; return cudaSuccess; }
template <typename K> cudaError_t set(K, cudaFuncAttribute, int bytes) {
  *limit = bytes;
  if (bytes == 200) rest(300);  // the larger one is slow to return
  return cudaSuccess;
}
#define cudaGetDevice current
#define cudaFuncSetAttribute set
#include "op_common.cuh"
int main() {
  std::atomic<int> at(0), seen[16] = {};
  limit = &at;
  std::thread large([&] { b2g::allow_smem(0, 200, seen); });
  std::thread small([&] { rest(100); b2g::allow_smem(0, 100, seen); });
  large.join();
  small.join();
  b2g::allow_smem(0, 200, seen);
  printf("%d %d\n", at.load(), seen[0].load());
}
"""


def test_a_smaller_size_does_not_come_behind_a_larger(tmp_path):
    (tmp_path / "limit.cu").write_text("#include <atomic>\n" + SRC)
    exe = str(tmp_path / "limit")
    subprocess.run(["nvcc", "-std=c++17", "-gencode", "arch=compute_100a,code=sm_100a", "-I",
                    os.path.join(PKG, "csrc"), "-o", exe, str(tmp_path / "limit.cu")], check=True)
    assert subprocess.run([exe], check=True, capture_output=True, text=True).stdout.split() == ["200", "200"]
