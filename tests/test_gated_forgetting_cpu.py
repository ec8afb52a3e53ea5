"""What the tests of forgetting hold the gated linear recurrence to: its recurrence in numpy's f32 keeps within the bounds, and a factor of
one, or one that forgets 5 % too much or too little, does not."""

import numpy as np
import pytest

from oracle import gated_oracle as O
from util_forgetting import CONSTANT, KEPT, rates


def f32_recurrence(S, rho, convex, wrong=1.0):
    """a from the rounded rest, as the kernels form it; runs of eight tokens joined, as they do; `wrong`: times what is forgotten."""
    f = np.float32
    rest = (-np.expm1(-rho)).astype(f)
    a = f(1) - f(wrong) * rest
    u = rest if convex else np.zeros_like(rest)
    A, H = np.ones_like(a), np.zeros_like(a)
    for _ in range(8):
        A, H = f(a * A), f(a * H + u)
    h = np.zeros_like(a) if convex else np.ones_like(a)
    for _ in range(S // 8):
        h = f(A * h + H)
    for _ in range(S % 8):
        h = f(a * h + u)
    return h.astype(np.float64)


@pytest.mark.parametrize("S,times", KEPT)
def test_bound_on_what_is_forgotten(S, times):
    rho = rates(S, times, 64)
    gone, bound = O.kept_state(S, rho)
    off = lambda wrong: np.abs(1 - f32_recurrence(S, rho, False, wrong) - gone) / gone  # noqa: E731
    assert (off(1.0) <= bound).all() and (bound < 0.02).all()
    for wrong in (0.0, 0.95, 1.05):
        assert (off(wrong) > bound).all(), wrong


@pytest.mark.parametrize("S,times", CONSTANT)
def test_bound_on_the_mean_of_a_constant(S, times):
    rho = rates(S, times, 64)
    value, bound = O.constant_input(S, rho)
    off = lambda wrong: np.abs(f32_recurrence(S, rho, True, wrong) - value) / value  # noqa: E731
    assert (off(1.0) <= bound).all() and (bound < 0.02).all()
    for wrong in (0.0, 0.95, 1.05):
        assert (off(wrong) > bound).all(), wrong


def test_closed_forms_are_those_of_the_recurrence():
    rho = np.array([1e-3, 0.05])
    one = np.ones((1, 500, 2))
    r = O.gated_scan(0 * one, 0 * one, rate=-2 * rho, h_initial=np.ones((1, 2)), input_scale="convex")
    assert np.allclose(1 - r["h_last"][0][0], O.kept_state(500, rho)[0], rtol=1e-12)
    r = O.gated_scan(one, 0 * one, rate=-2 * rho, input_scale="convex")
    assert np.allclose(r["h_last"][0][0], O.constant_input(500, rho)[0], rtol=1e-12)
