"""How a gated linear recurrence is cut into units (csrc/gated_units.h, plain numbers, compiled with the host compiler): every token of
every channel in one unit, scratch that holds what the kernels index; and the order in which units wait for one another, run by a model
of CTAs that take them by a counter and stop anywhere."""

import os
import random
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "mlstm_kernels_b200", "csrc")
PROGRAM = r"""
#include <cstdio>
#include "gated_units.h"
int main() {
  int B, S, D, slots, back;
  while (scanf("%d %d %d %d %d", &B, &S, &D, &slots, &back) == 5) {
    const mlstm::GatedPlan p = mlstm::gated_plan(B, S, D, slots);
    const mlstm::GatedScratch s = mlstm::gated_scratch(p, B, D, back != 0);
    printf("%d %d %d %d %d %lld %lld %zu %zu %zu %zu\n", p.blocks, p.warps, p.nt, p.group, p.groups, p.chains, p.units, s.state, s.agg, s.rate, s.bytes);
  }
}
"""
SIZES = [(1, 1, 1), (1, 8, 64), (3, 9, 65), (2, 64, 128), (2, 65, 128), (1, 72, 7), (1, 8077, 2048), (1, 65536, 2048), (8, 4096, 2048), (4, 8192, 4096),
         (3, 777, 1001), (700, 3, 64), (1, 1 << 20, 64), (521, 2048, 2048), (1, 1 << 30, 8), (16, 500, 100)]


@pytest.fixture(scope="module")
def plan(tmp_path_factory):
    d = tmp_path_factory.mktemp("units")
    (d / "plan.cpp").write_text(PROGRAM)
    subprocess.run(["g++", "-std=c++17", f"-I{CSRC}", str(d / "plan.cpp"), "-o", str(d / "plan")], check=True)
    names = ("blocks", "warps", "nt", "group", "groups", "chains", "units", "state", "agg", "rate", "bytes")

    def ask(*args):
        out = subprocess.run([str(d / "plan")], input=" ".join(str(int(a)) for a in args), capture_output=True, text=True, check=True).stdout
        return dict(zip(names, (int(v) for v in out.split())))
    return ask


@pytest.mark.parametrize("B,S,D", SIZES)
@pytest.mark.parametrize("slots", [2, 444])
def test_units_cover_everything_and_scratch_holds_them(plan, B, S, D, slots):
    for back in (0, 1):
        p = plan(B, S, D, slots, back)
        tile = 8 * p["warps"]
        assert 1 <= p["warps"] <= 7 and p["nt"] * tile >= S > (p["nt"] - 1) * tile
        assert p["blocks"] * 64 >= D > (p["blocks"] - 1) * 64
        assert p["chains"] == B * p["blocks"] and p["units"] == p["chains"] * p["nt"] < 1 << 31
        assert p["group"] in (1, 2, 4, 8, 16) and p["groups"] * p["group"] >= p["nt"] > (p["groups"] - 1) * p["group"]
        # a pair of channels to a lane: 8 bytes of a state, 16 of a run
        if p["nt"] > 1:
            assert p["state"] >= 256 and p["agg"] - p["state"] >= 32 * 8 * p["chains"] * p["groups"]
            assert p["rate"] - p["agg"] >= (32 * 16 * p["units"] if p["group"] > 1 else 0)
        else:
            assert p["group"] == 1 and p["rate"] == 0
        assert all(p[n] % 256 == 0 for n in ("state", "agg", "rate", "bytes"))
        assert p["bytes"] - p["rate"] >= (4 * B * p["nt"] * D if back else 0)


def run_units(chains, nt, group, ctas, rng, ahead=2):
    """CTAs that take units by a counter, `ahead` of them before they work on the first, and are stopped and resumed at random between
    any two accesses to what they share.  Returns the state in front of every unit; runs are functions h -> a h + b."""
    runs = {(c, k): (rng.choice((0.5, 2.0, -1.0)), float(rng.randrange(-3, 4))) for c in range(chains) for k in range(nt)}
    counter, state, published, start = [0], {}, {}, {}

    def take():
        counter[0] += 1
        return counter[0] - 1

    def cta():
        units = []
        for _ in range(ahead):
            units.append(take())
            yield
        while units[0] < chains * nt:
            k, c = divmod(units.pop(0), chains)
            units.append(take())
            yield
            g, pos = divmod(k, group)
            more, last = k < nt - 1, pos == group - 1
            if more and not last:
                published[c, k] = runs[c, k]
                yield
            while not ((g == 0 or (c, g) in state) and all((c, g * group + n) in published for n in range(pos))):
                yield "waits"
            h = 1.0 + c if g == 0 else state[c, g]
            for n in range(pos):
                a, b = published[c, g * group + n]
                h = a * h + b
                yield
            start[c, k] = h
            if more and last:
                a, b = runs[c, k]
                state[c, g + 1] = a * h + b
                yield
    alive = [cta() for _ in range(ctas)]
    idle = 0
    while alive:
        n = rng.randrange(len(alive))
        try:
            idle = idle + 1 if next(alive[n]) == "waits" else 0
        except StopIteration:
            alive.pop(n)
            idle = 0
        assert idle < 1000 * ctas, "every CTA waits"
    return runs, start


@pytest.mark.parametrize("chains,nt,group", [(1, 1, 1), (1, 7, 1), (3, 5, 1), (1, 33, 16), (2, 16, 16), (2, 17, 4), (5, 9, 2), (40, 3, 2), (1, 64, 8)])
@pytest.mark.parametrize("ctas", [1, 2, 3, 20])
def test_no_unit_waits_for_one_that_is_not_under_way(chains, nt, group, ctas):
    rng = random.Random(chains * 1000 + nt * 10 + ctas)
    for _ in range(5):
        runs, start = run_units(chains, nt, group, ctas, rng)
        for c in range(chains):
            h = 1.0 + c
            for k in range(nt):
                assert start[c, k] == h
                a, b = runs[c, k]
                h = a * h + b
