"""Registers and spills of the gated linear recurrence's and dropout's kernels, as the compiler reports them: as many CTAs to an SM as the
kernels' comments say, and no more spilled than the profile says.  And no field of a launch's sizes that nothing reads, which moves
registers about by where it puts the others."""

import glob
import os
import re

from test_kernel_registers import CSRC, pytestmark, report  # noqa: F401


def test_gated_scan():
    kernels, name = report("gated_scan_bf16.cu"), "__nv_bfloat16"
    fw = {n: x for n, x in kernels.items() if n.startswith("gated_fw_rows<")}
    bw = {n: x for n, x in kernels.items() if n.startswith("gated_bw_rows<")}
    assert len(fw) == len(bw) == 24
    # 256 threads: three CTAs of 80 registers, two of 128, to an SM of 65536
    assert max(r for r, _ in fw.values()) <= 80 and max(r for r, _ in bw.values()) <= 128
    # bytes stored and loaded
    assert max(s for _, s in fw.values()) <= 32 and max(s for _, s in bw.values()) <= 8
    # the backward with a rate has the most to hold
    assert all(s == 0 for n, (_, s) in bw.items() if "GatedFixed<true" in n)
    assert kernels[f"gated_fw_any<{name}>"] <= (128, 0)
    assert kernels[f"gated_bw_any<{name}>"][0] <= 128 and kernels[f"gated_bw_any<{name}>"][1] <= 248


def test_dropout():
    """Four CTAs of 256 threads to an SM; only two residuals of 16 bits take more registers than that leaves."""
    kernels = report("dropout.cu")
    wide = {n: x for n, x in kernels.items() if n.startswith("dropout_wide<")}
    assert len(wide) >= 20 and max(r for r, _ in wide.values()) <= 64
    spilled = {n: s for n, (_, s) in wide.items() if s > 0}
    assert all(re.search(r"<(__nv_bfloat16|__half), \1, 8, \w+, true>", n) for n in spilled) and max(spilled.values()) <= 208


def test_every_size_of_a_launch_is_read():
    with open(os.path.join(CSRC, "gated.cuh")) as f:
        src = f.read()
    body = re.search(r"struct GatedDims \{(.*?)\n\};", src, re.S).group(1)
    body = re.sub(r"//[^\n]*", "", body)
    fields = [n for decl in body.split(";") for n in re.findall(r"[\s*](\w+)\s*(?=,|$)", decl.strip())]
    assert {"looks", "S", "D", "nc", "gt", "agg", "gave_up"} <= set(fields)
    kernels = "".join(open(p).read() for p in glob.glob(os.path.join(CSRC, "gated*.cuh")))
    kernels = re.sub(r"//[^\n]*", "", kernels)
    assert [n for n in fields if not re.search(rf"\bq\.{n}\b", kernels)] == []
