"""How the expert products count the clusters a device holds, and cut their work by it.

The host code is compiled into small programs with nvcc; the first needs no GPU.
"""

import subprocess

import pytest

from loraforge_b200 import _build


def program(folder, body):
    source = folder / "program.cu"
    source.write_text('#include <cstdio>\n#include "grouped.cuh"\n'
                      "namespace lfb { std::string& last_error() { static std::string s; return s; } }\n"
                      "using namespace lfb::grouped;\n" + body)
    out = folder / "program"
    subprocess.run([_build.nvcc(), *_build.ARCH, "-O1", "-std=c++17", "--expt-relaxed-constexpr", "-I", str(_build.INCLUDE),
                    "-I", str(_build.CSRC), str(source), "-o", str(out)], check=True, capture_output=True)
    return out


CUTS = """
int main() {
  // Long contractions of few groups are split over many CTAs, here with nothing above `most` to hold them.
  for (int most = 1; most <= kMaxSplit; ++most) {
    Clusters c{};
    for (int s = 1; s <= most; ++s) c.at_once[s] = 148 / s;
    const Cut cut = choose_cut(c, 1, 256, 256, 1, true);
    std::printf("%d\\n", cut.split);
  }
  // What the device cannot place is an error of the call, not a grid of none.
  Clusters pairs{};
  pairs.at_once[2] = 74;
  return grid_of(pairs, 5, 2, "call") == 10 && grid_of(pairs, 500, 2, "call") == 148 && lfb::last_error().empty() &&
                 grid_of(pairs, 5, 4, "call") == 0 && lfb::last_error() == "call: the device cannot place a cluster of 4 CTAs"
             ? 0 : 3;
}
"""


def test_no_cut_over_more_ctas_than_a_cluster_may_have(tmp_path):
    out = subprocess.run([program(tmp_path, CUTS)], capture_output=True, text=True)
    assert out.returncode == 0, out.returncode
    splits = [int(v) for v in out.stdout.split()]
    assert all(1 <= split <= most for most, split in enumerate(splits, 1)) and splits[-1] > 1


COUNTS = """
__global__ void all_of_an_sm(int) {}
__global__ void little_of_an_sm(int) {}
int main() {
  int flags[64] = {};
  Clusters a{}, b{}, c{};
  if (lfb::ensure_smem(all_of_an_sm, 200 * 1024, flags)) return 1;
  if (clusters_of(all_of_an_sm, 128, 200 * 1024, &a) || clusters_of(little_of_an_sm, 128, 1024, &b) || clusters_of(all_of_an_sm, 128, 200 * 1024, &c)) return 2;
  std::printf("%d %d %d\\n", a.at_once[1], b.at_once[1], c.at_once[1]);
}
"""


@pytest.mark.gpu
def test_each_kernel_has_its_own_counts(tmp_path):
    torch = pytest.importorskip("torch")
    if not torch.cuda.is_available():
        pytest.skip("CUDA device required")
    out = subprocess.run([program(tmp_path, COUNTS)], capture_output=True, text=True)
    assert out.returncode == 0, out.returncode
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    assert [int(v) for v in out.stdout.split()][::2] == [sms, sms]  # 200 KB each: one a SM
    assert int(out.stdout.split()[1]) >= 4 * sms  # 128 threads and 1 KB each: many a SM
