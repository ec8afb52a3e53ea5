"""Calls from several Python threads at once (the native functions release the GIL before they launch)."""

import threading

import numpy as np
import pytest
import torch

import mlstm_kernels_b200 as mk
from mlstm_kernels_b200.recurrent import mlstm_recurrent_step__b200_fw
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


@pytest.mark.parametrize("backward", [False, True])
def test_portable_chunkwise_of_different_head_dims(backward):
    def job(DHQK):
        rng = np.random.default_rng(DHQK)
        t = [make(rng, 1, 2, 128, n, grad=backward) for n in (DHQK, DHQK, 32)] + [make(rng, 1, 2, 128, grad=backward) for _ in range(2)]

        def run():
            h = mk.mlstm_chunkwise__b200_xl_chunk(*t, chunk_size=64, impl="simt")
            return [h.detach(), *torch.autograd.grad(h, t, torch.ones_like(h))] if backward else [h]
        return run
    at_once([job(D) for D in (256, 32, 128, 64)], 100 if backward else 500)


def step_job(DHQK):
    rng = np.random.default_rng(DHQK)
    q, k, v = make(rng, 1, 1, DHQK), make(rng, 1, 1, DHQK), make(rng, 1, 1, 32)
    i, f, m = (make(rng, 1, 1, 1) for _ in range(3))
    c, n = make(rng, 1, 1, DHQK, 32), make(rng, 1, 1, DHQK)

    def run():   # (through the C interface, without the GIL)
        h, new = mlstm_recurrent_step__b200_fw(c, n, m, q, k, v, i, f, *(torch.empty_like(t) for t in (c, n, m)), vecH_out=torch.empty_like(v), validate=False)
        return [h, *new]
    return run


def test_steps_of_different_head_dims():
    """Beyond 6000 a step's operands need more shared memory than a kernel has unasked."""
    at_once([step_job(D) for D in (8192, 6400, 7168, 6144)], 500)


def test_step_between_the_limits_with_and_without_static_memory():
    """Head dims whose operands fit the 48 KB that a kernel has unasked, but not beside its static memory."""
    for D in (6008, 6012, 6016, 6020):
        h, c, n, m = step_job(D)()
        assert all(torch.isfinite(t).all() for t in (h, c, n, m)) and (n != 0).any()
