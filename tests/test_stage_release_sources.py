"""Shared memory that the TMA engine fills is given back to it by threads that have read it only behind a proxy fence: an arrival on an mbarrier
orders their reads before other threads' accesses, not before writes through the async proxy.  Checked in the sources."""

import os
import re

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "mlstm_kernels_b200", "csrc")
# barriers on which threads (not the tensor core's commits) give such memory back
RELEASES = {"chunkwise_sm100.cu": (r"warp_arrive\(&bar_empty\[", r"mbar_arrive\(&sh\.bar_qdone\[", r"mbar_arrive\(&sh\.bar_done\["),
            "chunkwise_bw_sm100.cu": (r"warp_arrive\(&sh\.staged\[",)}


def test_reads_are_fenced_before_a_stage_goes_back():
    for name, releases in RELEASES.items():
        with open(os.path.join(CSRC, name)) as f:
            src = re.sub(r"//[^\n]*", "", f.read())
        for release in releases:
            places = [m.start() for m in re.finditer(release, src)]
            assert places, release
            for at in places:
                before = src[:at].rstrip()
                between = before[before.rindex("fence_proxy_async_smem();"):]
                # nothing but the election of the arriving thread, or the test of the abort flag, in between
                rest = re.sub(r"fence_proxy_async_smem\(\);|__syncwarp\(\);|if \(lane == 0\)|if \(!aborted\(smem_u32\(&sh\.abort\)\)\)", "", between)
                assert rest.strip() == "", (name, release, rest)
