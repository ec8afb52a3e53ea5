"""How layer norm's kernels take a row (csrc/norm_rows.h, plain numbers), compiled with the host compiler: every width that is whole
chunks of 16 bytes is taken in chunks, and the threads' chunks cover every column once."""

import os
import subprocess

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "mlstm_kernels_b200", "csrc")
PROGRAM = r"""
#include <cstdio>
#include "norm_rows.h"
int main() {
  printf("%d %d\n", mlstm::LN_V, mlstm::LN_MAX_D);
  for (int d = 1; d <= mlstm::LN_MAX_D; ++d)
    printf("%d %d %d\n", mlstm::ln_threads(d), mlstm::ln_whole_chunks(d, 2), mlstm::ln_whole_chunks(d, 4));
}
"""


def test_rows_of_every_width(tmp_path):
    (tmp_path / "rows.cpp").write_text(PROGRAM)
    subprocess.run(["g++", "-std=c++17", f"-I{CSRC}", str(tmp_path / "rows.cpp"), "-o", str(tmp_path / "rows")], check=True)
    out = subprocess.run([str(tmp_path / "rows")], capture_output=True, text=True, check=True).stdout.split("\n")
    per_thread, most = map(int, out[0].split())
    assert most == 16384
    for d, line in zip(range(1, most + 1), out[1:]):
        threads, half, full = map(int, line.split())
        assert half == (d % 8 == 0) and full == (d % 4 == 0), d
        # as the kernels are compiled for; enough of them; at most one warp, or an eighth above 256 threads' worth, too many
        assert threads in (4, 8, 16, 32, 64, 96, 128, 160, 192, 224, 256, 512, 1024) and threads * per_thread >= d, d
        assert threads <= 4 or threads > 256 or threads < 2 * d / per_thread + 32, d
        for e in (8, 4):
            if d % e == 0:   # chunk q of thread t begins at column (q threads + t) e
                chunks = [(q * threads + t) * e for q in range(per_thread // e) for t in range(threads)]
                assert [c for c in chunks if c < d] == list(range(0, d, e)), d
