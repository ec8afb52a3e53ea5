"""Kernels' limits of dynamic shared memory when threads launch them with different sizes at once (csrc/smem_limits.h, plain C++, compiled
with the host compiler): no thread finds the limit below what it was granted, and a failed raise is not taken for done."""

import glob
import os
import re
import subprocess

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "mlstm_kernels_b200", "csrc")
PROGRAM = r"""
#include <atomic>
#include <cstdio>
#include <thread>
#include <vector>
#include "smem_limits.h"
int main() {
  mlstm::SmemLimits limits;
  static std::atomic<size_t> real[2][3];   // what a launch would be checked against, by device and kernel
  static int kernels[3];
  std::atomic<long> bad{0}, lowered{0}, sets{0};
  std::vector<std::thread> threads;
  for (int t = 0; t < 8; ++t)
    threads.emplace_back([&, t] {
      for (int n = 0; n < 20000; ++n) {
        const int dev = n & 1, k = (n + t) % 3;
        const size_t need = 1024 * (1 + (size_t)((n * 7 + t * 13) % 200));
        const int rc = limits.allow(dev, &kernels[k], need, [&] {
          if (real[dev][k].exchange(need) > need) ++lowered;
          ++sets;
          return 0;
        });
        if (rc != 0 || real[dev][k].load() < need) ++bad;   // the launch
      }
    });
  for (auto& t : threads) t.join();
  const int fails = limits.allow(5, &kernels[0], 4096, [] { return -6; }), again = limits.allow(5, &kernels[0], 4096, [] { return 0; });
  const int known = limits.allow(5, &kernels[0], 4096, [] { return -9; }), less = limits.allow(5, &kernels[0], 100, [] { return -9; });
  printf("%ld %ld %d %d %d %d %d\n", bad.load(), lowered.load(), sets.load() <= 6 * 200, fails, again, known, less);
}
"""


def test_no_thread_lowers_what_another_was_granted(tmp_path):
    (tmp_path / "limits.cpp").write_text(PROGRAM)
    subprocess.run(["g++", "-O2", "-std=c++17", "-pthread", f"-I{CSRC}", str(tmp_path / "limits.cpp"), "-o", str(tmp_path / "limits")], check=True)
    out = subprocess.run([str(tmp_path / "limits")], capture_output=True, text=True, check=True, timeout=120).stdout
    assert out.split() == ["0", "0", "1", "-6", "0", "0", "0"]


def sizes_set():
    """(file, text) of every place that sets a kernel's limit."""
    for path in sorted(glob.glob(os.path.join(CSRC, "*.cu*"))):
        with open(path) as f:
            for m in re.finditer(r"cudaFuncSetAttribute\((.*?)\)\)?;", f.read()):
                yield os.path.basename(path), m.group(1)


def test_gated_scan_takes_its_limit_from_there():
    """Its need goes by the number of warps, and so by the sequences' length."""
    assert not [name for name, _ in sizes_set() if name.startswith("gated")]
    with open(os.path.join(CSRC, "gated_tiles.cuh")) as f:
        assert "allow_smem((const void*)kern, smem)" in f.read()


def test_only_sizes_that_are_constants_of_a_kernel_are_set_elsewhere():
    """A size that is the same in every call of a kernel can be set by any thread at any time."""
    constant = {"tensor_maps.cuh", "layer_norm.cu", "short_conv.cu", "ssm.cuh"}   # (a kernel's template arguments give it)
    assert {name for name, _ in sizes_set()} == constant | {"api.cu"}
    for name in ("chunkwise_simt.cu", "step.cu"):
        with open(os.path.join(CSRC, name)) as f:
            assert "allow_smem((const void*)kern, smem)" in f.read(), name
    for name, call in (("layer_norm.cu", "ln_run"), ("short_conv.cu", "conv_bw_run"), ("ssm_fw.cu", "ssm_launch"), ("ssm_bw.cu", "ssm_launch")):
        with open(os.path.join(CSRC, name)) as f:
            src = f.read()
        calls = len(re.findall(rf"(?<!int ){call}\(\w+<", src))
        assert calls > 0 and len(re.findall(rf"(?<!int ){call}\(\w+<[^>]*>, [^;:]*\w+<[^>]*>::BYTES, ", src)) == calls, name
