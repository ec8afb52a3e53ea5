"""Waits of the gated linear recurrence that run out: in a model of its CTAs every one of them ends, whichever units nobody does; on the GPU
the call ends, the status word says so, and the next call is right."""

import random

import numpy as np
import pytest
import torch

import mlstm_kernels_b200 as mk
from mlstm_kernels_b200 import _lib


def run_with_units_left_out(chains, nt, group, ctas, left_out, limit, rng):
    """CTAs as in csrc/gated_tiles.cuh, stopped and resumed at random; a wait that has looked `limit` times, or finds that another has, goes on
    without.  Returns how many waits ran out, and the units that were done."""
    counter, state, published, done, gave_up = [left_out], set(), set(), set(), [0]

    def take():
        counter[0] += 1
        return counter[0] - 1

    def cta():
        units = [take(), take()]
        while units[0] < chains * nt:
            k, c = divmod(units.pop(0), chains)
            units.append(take())
            yield
            g, pos = divmod(k, group)
            more, last = k < nt - 1, pos == group - 1
            if more and not last:
                published.add((c, k))
            looks = 0
            while not ((g == 0 or (c, g) in state) and all((c, g * group + n) in published for n in range(pos))):
                looks += 1
                if gave_up[0] or looks >= limit:
                    gave_up[0] += looks >= limit
                    break
                yield
            done.add((c, k))
            if more and last:
                state.add((c, g + 1))
    alive = [cta() for _ in range(ctas)]
    for _ in range(200 * limit * (ctas + chains * nt)):
        if not alive:
            break
        n = rng.randrange(len(alive))
        try:
            next(alive[n])
        except StopIteration:
            alive.pop(n)
    assert not alive, "a CTA still waits"
    return gave_up[0], done


@pytest.mark.parametrize("chains,nt,group", [(1, 7, 1), (3, 5, 1), (1, 33, 16), (2, 17, 4), (5, 9, 2)])
@pytest.mark.parametrize("ctas", [1, 2, 20])
def test_every_cta_of_the_model_ends(chains, nt, group, ctas):
    rng = random.Random(chains * 1000 + nt * 10 + ctas)
    for left_out in (0, 1, chains, 2 * chains + 1, chains * nt - 1):
        ran_out, done = run_with_units_left_out(chains, nt, group, ctas, left_out, 10 ** 6 if left_out == 0 else 20, rng)
        assert len(done) == chains * nt - left_out
        # the last unit alone is in a chain whose others are left out, or has nothing in front of it
        assert (ran_out > 0) == (left_out > 0)


def test_limits_of_the_selftest():
    lib = _lib.load()
    for looks, units in ((0, 1), (256, 0), (256, -1), (256, 256), (1000001, 1)):
        assert lib.mlstm_b200_selftest_gated_wait_expiry(looks, units) == -7
    assert lib.mlstm_b200_selftest_gated_wait_expiry(256, 1) == 0 and lib.mlstm_b200_selftest_gated_wait_expiry(0, 0) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("B,S,D,units", [(1, 400, 64, 1), (2, 2000, 63, 3), (1, 30000, 128, 40), (40, 300, 96, 255)])
@pytest.mark.parametrize("rate", [False, True])
def test_a_wait_that_runs_out_is_reported(B, S, D, units, rate, dtype):
    from test_gated_gpu import inputs
    from util_layers import make
    name = {torch.float32: "f32", torch.bfloat16: "bf16", torch.float16: "f16"}[dtype]
    t = inputs(3, B, S, D, name, rate=rate, grad=False)
    lib, host = _lib.load(), _lib.host()
    args = [t.get(n) for n in ("x", "f", "i", "z", "rate", "h_initial")] + [1]
    dy, dh = make(np.random.default_rng(1), B, S, D, dtype=dtype), make(np.random.default_rng(2), B, D)
    y, last, ck = host.gated_scan_fw(*args, True, True)
    grads = host.gated_scan_bw(*args, ck, dy, dh)
    torch.cuda.synchronize()
    assert _lib.device_status() == 0
    for call in (lambda: host.gated_scan_fw(*args, True, True), lambda: host.gated_scan_bw(*args, ck, dy, dh)):
        assert lib.mlstm_b200_selftest_gated_wait_expiry(2048, units) == 0
        call()
        assert _lib.device_status(reset=False) == 301
        assert _lib.device_status() == 301 and _lib.device_status() == 0   # kept until it is cleared
        for got, want in zip((*host.gated_scan_fw(*args, True, True)[:2], *host.gated_scan_bw(*args, ck, dy, dh)), (y, last, *grads)):
            assert (got is None and want is None) or torch.equal(got, want)
        assert _lib.device_status() == 0
    # a sequence of one unit waits for nothing, and the request ends with it
    one = [v[:, :50] if v is not None and v.dim() == 3 else v for v in args[:6]] + [1]
    assert lib.mlstm_b200_selftest_gated_wait_expiry(2048, 1) == 0
    assert torch.equal(host.gated_scan_fw(*one, False, False)[0], mk.gated_scan__b200(*one[:6], input_scale="convex"))
    assert torch.equal(host.gated_scan_fw(*args, False, False)[0], y) and _lib.device_status() == 0
