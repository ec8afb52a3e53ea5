"""What a state of the gated linear recurrence forgets, and what a "convex" one comes to under a constant input, against closed forms: over one
token to some memories of channels that remember up to 65536 tokens.  (That a factor of one, or forgetting 5 % off, is found is tested on
the CPU.)"""

import numpy as np
import pytest
import torch

import mlstm_kernels_b200 as mk
from oracle import gated_oracle as O
from util_forgetting import CONSTANT, KEPT, rates
from util_layers import TDT, f64

pytestmark = pytest.mark.gpu


def gates(rho, dtype, rated):
    """f (D,), the rate (D,) or None, and the -log a that they stand for."""
    T = TDT[dtype]
    if rated:
        f = torch.full((len(rho),), -1.0, dtype=T, device="cuda")
        s = 1 / (1 + np.exp(1.0))
        rate = torch.from_numpy(-rho / s).float().cuda()
        return f, rate, -f64(rate) * s
    f = torch.from_numpy(-np.log(np.expm1(rho))).to(T).cuda()   # sigmoid(f) = e^-rho
    return f, None, np.log1p(np.exp(-f64(f)))


def run(S, times, D, dtype, rated, convex, one_by_one=False):
    f, rate, rho = gates(rates(S, times, D), dtype, rated)
    value, bound = (O.constant_input if convex else O.kept_state)(S, rho)
    x = torch.full((2, S, D), float(convex), dtype=TDT[dtype], device="cuda")
    h = torch.full((2, D), float(not convex), device="cuda")
    f = f.expand(2, S, D)
    if one_by_one:
        for t in range(S):
            _, h = mk.gated_step__b200(x[:, t], f[:, t], h, rate=rate, input_scale="convex", h_new=h)
    else:
        _, h = mk.gated_scan__b200(x, f, rate=rate, h_initial=h, return_last_states=True, input_scale="convex")
    got = f64(h) if convex else 1 - f64(h)
    assert (np.abs(got - value) <= bound * value).all(), (np.abs(got / value - 1) / bound).max()


FORMS = [(f, times, convex) for convex, cases in ((False, KEPT), (True, CONSTANT)) for f, times in cases]


@pytest.mark.parametrize("S,times,convex", FORMS)
@pytest.mark.parametrize("rated", [False, True])
@pytest.mark.parametrize("dtype", list(TDT))
@pytest.mark.parametrize("D", [64, 63])
def test_scan(D, dtype, rated, S, times, convex):
    run(S, times, D, dtype, rated, convex)


@pytest.mark.parametrize("S,times,convex", [c for c in FORMS if c[0] <= 1000])
@pytest.mark.parametrize("rated", [False, True])
def test_steps(rated, S, times, convex):
    run(S, times, 64, "bf16", rated, convex, one_by_one=True)
