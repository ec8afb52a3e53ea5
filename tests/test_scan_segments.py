"""The rule that cuts a sequence of the selective state space scan into segments (csrc/scan_segments.h, plain numbers), compiled with
the host compiler: against sizes that were timed with every number of segments on a GPU of 148 SMs."""

import os
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "mlstm_kernels_b200", "csrc")
PROGRAM = r"""
#include <cstdio>
#include "scan_segments.h"
int main() {
  long long ctas, own_ctas;
  int turns, nt, np, backward;
  unsigned long whole, own;
  while (scanf("%lld %d %lld %d %d %d %lu %lu", &ctas, &turns, &own_ctas, &nt, &np, &backward, &whole, &own) == 8) {
    const mlstm::ScanSlots held{mlstm::scan_resident(whole, backward ? 4 : 5), mlstm::scan_resident(own, 5)};
    printf("%d %d %d\n", mlstm::scan_segments(ctas, turns, own_ctas, nt, np, backward != 0, held, 148), held.whole, held.own);
  }
}
"""
# shared memory of a CTA by padded states and bytes of an element: forward, its own ends, backward, its own ends
SHARED = {(8, 2): (52224, 33792, 89152, 41984), (8, 4): (77824, 50688, 122944, 67072), (16, 2): (44032, 27648, 52288, 35840), (16, 4): (44032, 27648, 70720, 35840),
          (32, 2): (31744, 18432, 40000, 22528), (32, 4): (52224, 30720, 52288, 38912), (64, 2): (34816, 18432, 37952, 20480), (64, 4): (57344, 30720, 50240, 34816),
          (128, 2): (54784, 27648, 49216, 28672), (128, 4): (90624, 46080, 67648, 48128)}
# B, S, D, N, bytes of an element: {segments: (us forward, us backward)}
TIMED = {
    (4, 2048, 2048, 8, 2): "9:144/385 1:312/1130 2:351/753 3:295/631 4:255/457 5:233/564 6:202/528 8:151/394 10:149/438 12:136/384 16:130/369 26:137/376 32:143/377 43:153/407 64:186/455",
    (4, 2048, 2048, 8, 4): "9:178/- 1:338/958 2:352/749 3:296/809 4:241/632 5:255/695 6:239/612 8:188/611 10:184/580 12:173/574 16:172/536 26:180/569 32:189/580 43:208/624 64:255/710",
    (4, 2048, 2048, 16, 2): "9:-/540 11:196/- 1:294/1777 2:412/1186 3:352/810 4:270/615 5:210/703 6:210/618 8:198/533 10:193/567 12:195/533 16:190/521 26:205/537 32:214/542 43:236/568 64:295/639",
    (4, 2048, 2048, 16, 4): "11:213/- 1:313/1435 2:446/1010 3:376/691 4:289/748 5:226/672 6:228/609 8:213/596 10:211/566 12:210/578 16:207/561 26:221/582 32:230/591 43:251/626 64:307/707",
    (4, 2048, 2048, 64, 2): "1:643/4210 2:705/2471 3:728/2811 4:689/2367 5:703/2508 6:720/2404 8:715/2355 10:726/2305 12:736/2302 16:749/2256 26:807/2254 32:849/2288 43:934/2357 64:1135/2587",
    (4, 2048, 2048, 128, 2): "1:1453/12516 2:1726/6958 3:1801/8682 4:1773/6974 5:1823/7495 6:1856/7076 8:1871/6975 10:1898/6820 12:1943/6719 16:1959/6536 26:2154/6331 32:2265/6346 43:2517/6451 64:3035/6860",
    (4, 2048, 2048, 128, 4): "1:2303/11636 2:2378/11517 3:2579/8433 4:2557/9200 5:2650/7851 6:2663/8367 8:2700/8099 10:2758/7923 12:2812/7896 16:2884/7912 26:3152/7258 32:3301/7115 43:3695/7051 64:4601/7492",
    (1, 16384, 1024, 8, 2): "37:-/426 54:184/- 1:2451/9203 2:1971/6175 3:1321/4127 4:993/3104 5:796/2502 6:667/2246 8:501/1675 10:501/1294 12:469/1156 16:438/908 20:376/757 26:307/593 32:280/480 43:225/538 64:161/412",
    (1, 16384, 1024, 8, 4): "37:206/566 1:2524/7506 2:2036/5533 3:1363/3728 4:1065/2785 5:858/2241 6:743/1894 8:660/1428 10:539/1153 12:505/977 16:365/746 20:365/964 26:240/759 32:244/638 43:250/673 64:199/629",
    (1, 16384, 1024, 64, 2): "18:-/2105 23:753/- 1:3240/13562 2:2449/8816 3:2275/6096 4:1828/4625 5:1671/3754 6:1425/3183 8:1077/2448 10:814/2712 12:931/2445 16:822/2161 20:795/2281 26:790/2103 32:756/2110 43:767/2089 64:780/2091",
    (1, 512, 1024, 8, 4): "1:82/234 2:69/158 3:50/114 4:40/89 5:36/99 6:34/102 8:27/82 16:20/81 32:18/81",
    (1, 512, 1024, 16, 2): "1:68/249 2:58/156 3:41/128 4:34/88 5:30/83 6:31/84 8:30/88 16:23/86 32:22/81",
    (1, 512, 1024, 128, 2): "1:152/1118 2:133/682 3:113/447 4:87/379 5:85/342 6:99/288 8:88/220 16:98/210 32:128/250",
    (1, 512, 1024, 128, 4): "11:-/247 1:150/1005 2:131/608 3:141/439 4:113/338 5:112/287 6:126/255 8:123/290 16:133/259 32:189/281",
}


def padded(N):
    return next(n for n in (8, 16, 32, 64, 128) if N <= n)


@pytest.fixture(scope="module")
def rule(tmp_path_factory):
    d = tmp_path_factory.mktemp("scan")
    (d / "rule.cpp").write_text(PROGRAM)
    subprocess.run(["g++", "-std=c++17", f"-I{CSRC}", str(d / "rule.cpp"), "-o", str(d / "rule")], check=True)

    def ask(B, S, D, N, size, backward):
        np_ = padded(N)
        tiles = -(-D * np_ // 1024)                            # CTAs of 1024 states
        turns = -(-tiles // 64) if backward else 1
        shared = SHARED[np_, size][2 * backward:2 * backward + 2]
        line = f"{B * -(-tiles // turns)} {turns} {B * tiles} {-(-S // 16)} {np_} {int(backward)} {shared[0]} {shared[1]}"
        return tuple(map(int, subprocess.run([str(d / "rule")], input=line, capture_output=True, text=True, check=True).stdout.split()))
    return ask


def table(text, backward):
    pairs = ((int(n), us.split("/")[backward]) for n, us in (item.split(":") for item in text.split()))
    return {n: int(us) for n, us in pairs if us != "-"}


@pytest.mark.parametrize("backward", [False, True])
@pytest.mark.parametrize("size", TIMED)
def test_number_of_segments_is_near_the_fastest(rule, size, backward):
    """The number that is taken was timed, and took at most 15 % longer than the fastest."""
    n, _, _ = rule(*size, backward)
    times = table(TIMED[size], backward)
    assert times[n] <= 1.15 * min(times.values()), (n, times[n], min(times.values()))


def test_resident_ctas(rule):
    """What 228 KB of shared memory hold: two CTAs of the backward and one in f32 with up to 8 states, three in f32 with 9 to 16 and 65 to 128."""
    held = {(n, size): [rule(1, 16, 8, n, size, b)[1:] for b in (False, True)] for n, size in SHARED}
    assert {k: v[1][0] for k, v in held.items() if v[1][0] < 4} == {(8, 2): 2, (8, 4): 1, (16, 4): 3, (128, 4): 3}
    assert {k: v[0][0] for k, v in held.items() if v[0][0] < 5} == {(8, 2): 4, (8, 4): 2, (32, 4): 4, (64, 4): 4, (128, 2): 4, (128, 4): 2}
