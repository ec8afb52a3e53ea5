"""Recurrences whose state goes from call to call in one buffer, as in training on pieces of longer texts: the buffer takes the next state
before the backward of the call that read it runs."""

import numpy as np
import pytest
import torch

import mlstm_kernels_b200 as mk
from mlstm_kernels_b200 import _ops
from test_gated_gpu import inputs
from util_layers import make

pytestmark = pytest.mark.gpu


def gated_traced(x, f, i, z, rate, h_initial, want_last):
    y, last, _ = _ops.gated_scan(x, f, i, z, rate, h_initial, 2, True, want_last)
    return (y, last) if want_last else y


def gated_eager(x, f, i, z, rate, h_initial, want_last):
    return mk.gated_scan__b200(x, f, i, z, rate, h_initial, want_last, "variance")


def written_over(fn, t, state, wants, shape):
    dy = make(np.random.default_rng(1), *shape, dtype=torch.bfloat16)
    h0 = t.pop("h_initial").detach().to(state)
    leaves = list(t.values())
    keep = h0.clone().requires_grad_(wants)
    want = torch.autograd.grad(fn(**t, h_initial=keep, want_last=False), [*leaves, *([keep] if wants else [])], dy)
    leaf = h0.clone().requires_grad_(wants)
    buffer = leaf.clone()   # (a leaf itself is not written to)
    y, last = fn(**t, h_initial=buffer, want_last=True)
    with torch.no_grad():
        buffer.copy_(last)
    got = torch.autograd.grad(y, [*leaves, *([leaf] if wants else [])], dy)
    for a, b in zip(want, got):
        assert a.dtype == b.dtype and torch.equal(a, b)
    if wants:
        assert got[-1].dtype == state and (got[-1] != 0).any()


@pytest.mark.parametrize("fn", [gated_eager, gated_traced, torch.compile(gated_eager, fullgraph=True)], ids=["eager", "operator", "compiled"])
@pytest.mark.parametrize("state", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("wants", [False, True])
def test_gated_scan(fn, state, wants):
    written_over(fn, inputs(7, 2, 130, 40, "bf16"), state, wants, (2, 130, 40))


def ssm_traced(x, dt, a, b, c, h_initial, want_last):
    y, last, _ = _ops.ssm_scan(x, dt, a, b, c, None, None, None, True, h_initial, True, want_last)
    return (y, last) if want_last else y


def ssm_eager(x, dt, a, b, c, h_initial, want_last):
    return mk.ssm_scan__b200(x, dt, a, b, c, h_initial=h_initial, return_last_states=want_last, softplus=True)


@pytest.mark.parametrize("fn", [ssm_eager, ssm_traced, torch.compile(ssm_eager, fullgraph=True)], ids=["eager", "operator", "compiled"])
@pytest.mark.parametrize("state", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("wants", [False, True])
def test_ssm_scan(fn, state, wants):
    rng = np.random.default_rng(8)
    m = lambda *s, **k: make(rng, *s, grad=True, **k)  # noqa: E731
    bf16 = dict(dtype=torch.bfloat16)
    t = dict(x=m(2, 130, 40, **bf16), dt=m(2, 130, 40, **bf16), a=(-torch.exp(make(rng, 40, 16))).requires_grad_(True), b=m(2, 130, 16, **bf16),
             c=m(2, 130, 16, **bf16), h_initial=m(2, 40, 16))
    written_over(fn, t, state, wants, (2, 130, 40))
