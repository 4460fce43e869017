"""The shared-memory limit of a kernel under host threads that raise it at once (no GPU).

The helper is compiled with nvcc into a small program in which the runtime's two calls are stand-ins.
"""

import subprocess

from loraforge_b200 import _build

SOURCE = """
#include <cuda_runtime.h>
#include <chrono>
#include <thread>
static int limit = 0;  // what the runtime holds for the kernel
static cudaError_t set_limit(void*, cudaFuncAttribute what, int value) {
  if (what == cudaFuncAttributeMaxDynamicSharedMemorySize) {
    // The lower of two requests is the slow one.
    if (value == 100 * 1024) std::this_thread::sleep_for(std::chrono::milliseconds(300));
    limit = value;
  }
  return cudaSuccess;
}
static cudaError_t first_device(int* device) { return *device = 0, cudaSuccess; }
#define cudaFuncSetAttribute set_limit
#define cudaGetDevice first_device
#include "launch.cuh"
namespace lfb { std::string& last_error() { static thread_local std::string s; return s; } }

int main() {
  int flags[64] = {}, a = 1, b = 1;
  void* kernel = nullptr;
  std::thread low([&] { a = lfb::ensure_smem(kernel, 100 * 1024, flags); });
  std::this_thread::sleep_for(std::chrono::milliseconds(100));
  std::thread high([&] { b = lfb::ensure_smem(kernel, 200 * 1024, flags); });
  low.join(), high.join();
  if (a || b) return 1;
  if (limit != 200 * 1024) return 2;
  return lfb::ensure_smem(kernel, 150 * 1024, flags) || limit != 200 * 1024 ? 3 : 0;
}
"""


def test_a_lower_limit_never_follows_a_higher_one(tmp_path):
    source, out = tmp_path / "program.cu", tmp_path / "program"
    source.write_text(SOURCE)
    subprocess.run([_build.nvcc(), *_build.ARCH, "-O1", "-std=c++17", "--expt-relaxed-constexpr", "-I", str(_build.INCLUDE),
                    "-I", str(_build.CSRC), str(source), "-o", str(out), "-lpthread"], check=True, capture_output=True)
    assert subprocess.run([out]).returncode == 0
