"""Calls from several Python threads at once (the native functions release the GIL before they launch)."""

import threading

import numpy as np
import pytest
import torch

import mlstm_kernels_b200 as mk
from util_layers import make

pytestmark = pytest.mark.gpu


def at_once(jobs, times):
    """Every job in a thread and a stream of its own, `times` times; what they gave, against what each gives alone."""
    alone = [job() for job in jobs]
    torch.cuda.synchronize()
    start, wrong = threading.Barrier(len(jobs)), []

    def work(job, want):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                start.wait(60)
                got = [job() for _ in range(times)]
                torch.cuda.current_stream().synchronize()
            for g in got:
                if not all(torch.equal(a, b) for a, b in zip(g, want)):
                    wrong.append("values")
                    return
        except Exception as e:  # noqa: BLE001
            wrong.append(repr(e))
    threads = [threading.Thread(target=work, args=a) for a in zip(jobs, alone)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert wrong == []


@pytest.mark.parametrize("backward", [False, True])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_gated_scans_of_different_lengths(dtype, backward):
    """The same kernels, which need shared memory by the sequences' length."""
    def job(S):
        rng = np.random.default_rng(S)
        t = [make(rng, 2, S, 64, dtype=dtype, grad=backward) for _ in range(4)]

        def run():
            y = mk.gated_scan__b200(*t, input_scale="convex")
            return [y.detach(), *torch.autograd.grad(y, t, torch.ones_like(y))] if backward else [y]
        return run
    at_once([job(S) for S in (56, 32, 48, 40)], 200 if backward else 1000)


def test_dropout():
    def job(n):
        x = make(np.random.default_rng(n), 300 + n, 1024, dtype=torch.bfloat16)
        return lambda: [mk.dropout__b200(x, 0.3, n, n)]
    at_once([job(n) for n in range(4)], 200)
