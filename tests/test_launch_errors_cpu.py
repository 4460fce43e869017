"""A launch that fails leaves no error behind for the next call's check (no GPU).

The launch helper is compiled with nvcc into a small program in which the runtime's calls are stand-ins:
a launch that fails, and the error that the runtime keeps until it is asked for.
"""

import subprocess

from loraforge_b200 import _build

SOURCE = """
#include <cuda_runtime.h>
static cudaError_t kept = cudaSuccess;
template <typename... T>
static cudaError_t failing_launch(T...) { return kept = cudaErrorInvalidConfiguration; }
static cudaError_t take() {
  const cudaError_t err = kept;
  kept = cudaSuccess;
  return err;
}
#define cudaLaunchKernelEx failing_launch
#define cudaGetLastError take
#include "grouped.cuh"
namespace lfb { std::string& last_error() { static std::string s; return s; } }
__global__ void nothing(int) {}
int main() {
  if (lfb::grouped::launch_clusters(nothing, 1, 4096, 1, 0, nullptr, "call", 1) != LF_E_CUDA) return 1;
  if (lfb::last_error().rfind("call: ", 0) != 0) return 2;
  return lfb::check_launch("the next call") == LF_OK ? 0 : 3;
}
"""


def test_the_next_call_does_not_see_the_error(tmp_path):
    source, out = tmp_path / "program.cu", tmp_path / "program"
    source.write_text(SOURCE)
    subprocess.run([_build.nvcc(), *_build.ARCH, "-O1", "-std=c++17", "--expt-relaxed-constexpr", "-I", str(_build.INCLUDE),
                    "-I", str(_build.CSRC), str(source), "-o", str(out)], check=True, capture_output=True)
    assert subprocess.run([out]).returncode == 0
