"""The operators around a recurrence in traced models: what their custom operators say of their outputs is what they return, the
gradient of heads comes back in the heads' layout, inference keeps nothing for a backward, and steps write the buffer they are given."""

import numpy as np
import pytest
import torch

import mlstm_kernels_b200 as mk
from mlstm_kernels_b200 import _lib
from util_layers import make

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16
OPS = torch.ops.mlstm_b200


def layouts(rng, D=40):
    """x (2, 5, 3, D) in several layouts."""
    return {"plain": make(rng, 2, 5, 3, D, dtype=BF16), "heads": make(rng, 2, 3, 5, D, dtype=BF16).transpose(1, 2),
            "slice": make(rng, 2, 5, 3, 100, dtype=BF16)[..., 8:8 + D], "expanded": make(rng, 1, 5, 3, D, dtype=BF16).expand(2, 5, 3, D),
            "last_axis": make(rng, 2, 5, D, 3, dtype=BF16).transpose(2, 3), "permuted": make(rng, 3, 2, 5, D, dtype=BF16).permute(1, 2, 0, 3)}


@pytest.mark.parametrize("how", ["plain", "heads", "slice", "expanded", "last_axis", "permuted"])
def test_norm_says_what_it_returns(how):
    rng = np.random.default_rng(1)
    x = layouts(rng)[how]
    w = make(rng, 3, 40)
    test = ("test_schema", "test_faketensor")
    torch.library.opcheck(OPS.layer_norm, (x, w, w, 1e-6), test_utils=test)
    _, mean, rstd = OPS.layer_norm(x, w, w, 1e-6)
    args = (x, w, mean, rstd, make(rng, 2, 5, 3, 40, dtype=BF16), True, torch.float32)
    torch.library.opcheck(OPS.layer_norm_bw, args, test_utils=test)
    if how in ("plain", "heads", "permuted"):
        assert OPS.layer_norm_bw(*args)[0].stride() == x.stride()


def test_heads_gradient_in_their_layout():
    rng = np.random.default_rng(2)
    h, w = make(rng, 2, 3, 50, 64, dtype=BF16, grad=True), make(rng, 3, 64, grad=True)
    dy = make(rng, 2, 50, 3, 64, dtype=BF16)
    fn = lambda h, w: mk.layer_norm__b200(h.transpose(1, 2), w)  # noqa: E731
    eager = torch.autograd.grad(fn(h, w), (h, w), dy)
    traced = torch.autograd.grad(torch.compile(fn, fullgraph=True)(h, w), (h, w), dy)
    assert traced[0].is_contiguous()
    for a, b in zip(eager, traced):
        assert torch.equal(a, b)


def scan_args(rng, S=200, D=32, N=16):
    m = lambda *s: make(rng, *s, dtype=BF16)  # noqa: E731
    return [m(2, S, D), m(2, S, D), -torch.exp(make(rng, D, N)), m(2, S, N), m(2, S, N)]


@pytest.mark.parametrize("keep", [False, True])
@pytest.mark.parametrize("want_last", [False, True])
def test_scan_says_what_it_returns(keep, want_last):
    t = scan_args(np.random.default_rng(3))
    args = (*t, None, None, None, True, None, keep, want_last)
    torch.library.opcheck(OPS.ssm_scan, args, test_utils=("test_schema", "test_faketensor"))
    y, h, ck = OPS.ssm_scan(*args)
    assert ck.numel() == (_lib.load().mlstm_b200_ssm_checkpoint_bytes(2, 200, 32, 16) if keep else 0)
    assert h.shape == ((2, 32, 16) if want_last else (0,))
    ref, last = mk.ssm_scan__b200(*t, softplus=True, return_last_states=True)
    assert torch.equal(y, ref) and (not want_last or torch.equal(h, last))


@pytest.mark.parametrize("want_last", [False, True])
def test_traced_inference_keeps_nothing(want_last):
    """No checkpoints, and no last state that nobody asked for: a traced call has no more memory at its peak than an eager one."""
    rng = np.random.default_rng(4)
    t = scan_args(rng, S=4096, D=256)
    fn = lambda *t: mk.ssm_scan__b200(*t, softplus=True, return_last_states=want_last)  # noqa: E731
    traced = torch.compile(fn, fullgraph=True)
    checkpoints = _lib.load().mlstm_b200_ssm_checkpoint_bytes(2, 4096, 256, 16)
    peaks = []
    for f in (fn, traced):
        f(*t)
        torch.cuda.synchronize()
        start = torch.cuda.memory_allocated()
        torch.cuda.reset_peak_memory_stats()
        out = f(*t)
        torch.cuda.synchronize()
        peaks.append(torch.cuda.max_memory_allocated() - start)
        del out
    assert abs(peaks[1] - peaks[0]) < checkpoints // 2, (peaks, checkpoints)
    leaf = [v.detach().requires_grad_(True) for v in t]   # and with a gradient it keeps them
    dy = make(rng, 2, 4096, 256, dtype=BF16)
    first = lambda r: r[0] if want_last else r  # noqa: E731
    for a, b in zip(torch.autograd.grad(first(fn(*leaf)), leaf, dy), torch.autograd.grad(first(traced(*leaf)), leaf, dy)):
        assert torch.equal(a, b)


def test_gradient_of_a_scan_that_kept_nothing_is_refused():
    t = [v.requires_grad_(True) for v in scan_args(np.random.default_rng(5))]
    y, _, _ = OPS.ssm_scan(*t, None, None, None, True, None, False, False)
    with pytest.raises(RuntimeError, match="checkpoints"):
        y.sum().backward()


def step_inputs(rng, B=3, D=40, N=16):
    x, s, w = make(rng, B, D, dtype=BF16), make(rng, B, 3, D, dtype=BF16), make(rng, D, 4)
    return x, s, w, -torch.exp(make(rng, D, N)), make(rng, B, N, dtype=BF16), make(rng, B, D, N)


@pytest.mark.parametrize("where", ["in place", "apart"])
def test_steps_with_buffers_compile(where):
    """A decode loop over fixed buffers, without a break of the graph: in place, and from one buffer to another and back."""
    x, s, w, a, b, h = step_inputs(np.random.default_rng(6))

    def steps(x, s, s2, h, h2):
        out = []
        for _ in range(2):
            u, r = mk.short_conv_step__b200(x, s, w, activation="silu", state_new=s2)
            y, g = mk.ssm_step__b200(u, x, a, b, b, h, softplus=True, h_new=h2)
            assert r is s2 and g is h2
            out.append(y)
            s, s2, h, h2 = s2, s, h2, h
        return out

    results = []
    for f in (steps, torch.compile(steps, fullgraph=True)):
        st, ht = s.clone(), h.clone()
        st2, ht2 = (st, ht) if where == "in place" else (torch.empty_like(st), torch.empty_like(ht))
        out = []
        for _ in range(3):
            out += f(x, st, st2, ht, ht2)
        results.append([*out, st, st2, ht, ht2])
    for p, q in zip(*results):
        assert torch.equal(p, q)


def test_steps_with_buffers_say_what_they_write():
    x, s, w, a, b, h = step_inputs(np.random.default_rng(7))
    test = ("test_schema", "test_faketensor")
    torch.library.opcheck(OPS.short_conv_step_into, (x, s, w, None, True, torch.empty_like(s)), test_utils=test)
    torch.library.opcheck(OPS.ssm_step_into, (x, x, a, b, b, h, None, None, None, True, torch.empty_like(h)), test_utils=test)
    y, new = mk.ssm_step__b200(x, x, a, b, b, h, softplus=True)
    buf = torch.empty_like(h)
    assert torch.equal(OPS.ssm_step_into(x, x, a, b, b, h, None, None, None, True, buf), y) and torch.equal(buf, new)
