"""The operators around a recurrence on the GPU where values grow, vanish or end a type's range, against the oracle in float64."""

import numpy as np
import pytest
import torch

import mlstm_kernels_b200 as mk
from oracle import layers_oracle as O
from util_layers import TDT, check, f64, make

pytestmark = pytest.mark.gpu


def scan(t, softplus, dy, dh):
    """y, the last state and all gradients against the oracle's."""
    ref = O.ssm_scan(**{n: f64(v) for n, v in t.items()}, softplus=softplus, dy=f64(dy), dh_last=f64(dh), summed=t["x"].shape[1])
    y, h = mk.ssm_scan__b200(**t, softplus=softplus, return_last_states=True)
    check(y, ref["y"], "y")
    check(h, ref["h_last"], "h_last")
    outs, ups = ((y, h), (dy, dh)) if dh is not None else ((y,), (dy,))
    for n, g in zip(t, torch.autograd.grad(outs, list(t.values()), ups)):
        check(g, ref["d" + n], "d" + n)
    return y, h


# Rates and steps above zero: a state is multiplied by e^6 with each token, by e^96 (more than f32 holds) with sixteen of them.
def growing(rng, B, S, D, N, dtype):
    T = TDT[dtype]
    bc = lambda: make(rng, B, S, N, dtype=T, grad=True)  # noqa: E731
    return dict(x=torch.zeros(B, S, D, dtype=T, device="cuda"), dt=torch.ones(B, S, D, dtype=T, device="cuda"),
                a=torch.full((D, N), 6.0, device="cuda"), b=bc(), c=bc())


@pytest.mark.parametrize("B,S,D,N", [(1, 600, 8, 4), (2, 401, 70, 16), (1, 350, 12, 64), (1, 40, 8, 16), (3, 1500, 64, 5)])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("gate", [False, True])
def test_zeros_in_front_of_a_state_that_grows(B, S, D, N, dtype, gate):
    """Inputs in the last twelve tokens, gradients in the first twelve: what comes from nothing stays nothing, however the sequence is cut."""
    rng = np.random.default_rng(S)
    t = growing(rng, B, S, D, N, dtype)
    T = TDT[dtype]
    t["x"][:, -12:] = make(rng, B, 12, D, dtype=T)
    if gate:
        t["z"] = make(rng, B, S, D, dtype=T)
    dy = torch.zeros(B, S, D, dtype=T, device="cuda")
    dy[:, :12] = make(rng, B, 12, D, dtype=T)
    scan({n: v.detach().requires_grad_(True) for n, v in t.items()}, False, dy, None)


@pytest.mark.parametrize("B,S,D,N", [(1, 600, 8, 4), (2, 401, 70, 16), (1, 350, 12, 64)])
@pytest.mark.parametrize("first", [16, 64, 160])
def test_a_small_state_that_grows(B, S, D, N, first):
    """Sixteen tokens that multiply a state of 2^-100 by e^96, nothing before and behind them; the last state's gradient likewise."""
    rng = np.random.default_rng(first)
    t = growing(rng, B, S, D, N, "f32")
    t["dt"].zero_()
    t["dt"][:, first:first + 16] = 1
    t["h_initial"] = make(rng, B, D, N, scale=2.0 ** -100)
    scan({n: v.detach().requires_grad_(True) for n, v in t.items()}, False, torch.zeros_like(t["x"]), make(rng, B, D, N, scale=2.0 ** -100))


def test_a_state_that_shrinks_out_of_a_segment_and_stays():
    """A state of 2^100 times e^-96: its decay alone is below what f32 holds, their product is not."""
    rng = np.random.default_rng(5)
    t = growing(rng, 1, 600, 8, 4, "f32")
    t["a"].fill_(-6.0)
    t["dt"].zero_()
    t["dt"][:, 16:32] = 1
    t["h_initial"] = make(rng, 1, 8, 4, scale=2.0 ** 100)
    dy = torch.zeros_like(t["x"])
    dy[:, 400:] = make(rng, 1, 200, 8)
    scan({n: v.detach().requires_grad_(True) for n, v in t.items()}, False, dy, make(rng, 1, 8, 4, scale=2.0 ** 100))


@pytest.mark.parametrize("S", [16, 17, 40, 601])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_rates_at_the_end_of_the_range(S, dtype):
    """States that forget everything at once, by rates near the lowest f32: behind the last token they still are what they were."""
    rng = np.random.default_rng(S)
    B, D, N, T = 2, 12, 8, TDT[dtype]
    m = lambda *s, **k: make(rng, *s, grad=True, **k)  # noqa: E731
    t = dict(x=m(B, S, D, dtype=T), dt=m(B, S, D, dtype=T), a=-torch.exp(make(rng, D, N)), b=m(B, S, N, dtype=T), c=m(B, S, N, dtype=T), z=m(B, S, D, dtype=T),
             h_initial=m(B, D, N))
    t["a"][:, ::3] = -3e38
    t["a"][2] = torch.finfo(torch.float32).min
    t["a"].requires_grad_(True)
    y, h = scan(t, True, make(rng, B, S, D, dtype=T), make(rng, B, D, N))
    with torch.no_grad():   # the plain -inf: a factor of zero
        a = t["a"].clone()
        a[2] = -float("inf")
        y2, h2 = mk.ssm_scan__b200(**{**t, "a": a}, softplus=True, return_last_states=True)
    assert torch.equal(y, y2) and torch.equal(h, h2)
