"""Dropout without a stored mask on the GPU: the mask against the generator restated in numpy, element by element, and the values against
float64; and a residual block of a recurrent layer with it."""

import ctypes

import numpy as np
import pytest
import torch

import mlstm_kernels_b200 as mk
from mlstm_kernels_b200 import _lib
from oracle import gated_oracle as O
from util_layers import TDT, check, f64, make

pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32
PAIRS = [("f32", None), ("bf16", None), ("f16", None), ("f32", "f32"), ("bf16", "bf16"), ("f16", "f16"), ("bf16", "f32"), ("f16", "f32")]
SEED, OFFSET = 0x1234567890ABCDEF, (7 << 32) + 11


def case(x, residual, p=0.3, seed=SEED, offset=OFFSET, dy=None):
    y = mk.dropout__b200(x, p, seed, offset, residual)
    out = x.dtype if residual is None else residual.dtype
    assert y.dtype == out and y.shape == x.shape and y.is_contiguous()
    dy = make(np.random.default_rng(1), *x.shape, dtype=out) if dy is None else dy
    number = int(seed.item()) if isinstance(seed, torch.Tensor) else seed
    ref = O.dropout(f64(x), p, number, offset, f64(residual), f64(dy))
    check(y, ref["y"], "y")
    keep = torch.from_numpy(O.kept(x.shape, p, number, offset)).cuda()
    if residual is None:
        assert torch.equal(y != 0, keep & (x != 0))
    leaves = [t for t in (x, residual) if t is not None and t.requires_grad]
    if leaves:
        grads = torch.autograd.grad(y, leaves, dy)
        for t, g in zip(leaves, grads):
            assert g.dtype == t.dtype
            check(g, ref["dx" if t is x else "dresidual"], "gradient")
        if x.requires_grad:
            assert torch.equal(grads[0] != 0, keep & (dy != 0))
            return grads[0]


@pytest.mark.parametrize("n", [1, 2, 3, 4, 5, 7, 8, 9, 15, 16, 17, 31, 33, 255, 256, 1023, 1025, 2047, 2049, 4095, 4097, 8192, 100003])
@pytest.mark.parametrize("dtype,residual", PAIRS)
def test_lengths(n, dtype, residual):
    rng = np.random.default_rng(n)
    case(make(rng, n, dtype=TDT[dtype], grad=True), None if residual is None else make(rng, n, dtype=TDT[residual], grad=True))


@pytest.mark.parametrize("shape", [(3, 37, 64), (2, 5, 1001), (7,), (), (2, 1, 3, 1, 5, 8), (1, 1), (4, 8, 2, 40)])
@pytest.mark.parametrize("p", [0.0, 1e-9, 0.1, 0.5, 0.999, 1.0])
def test_shapes_and_probabilities(shape, p):
    rng = np.random.default_rng(2)
    for dtype, residual in (("bf16", "f32"), ("f32", None)):
        case(make(rng, *shape, dtype=TDT[dtype], grad=True), None if residual is None else make(rng, *shape, dtype=TDT[residual], grad=True), p)


@pytest.mark.parametrize("how", ["heads", "slice", "offset", "odd_slice", "expanded", "last_axis", "six_axes", "residual_apart"])
@pytest.mark.parametrize("D", [40, 33])
def test_strides(how, D):
    """The mask goes by an element's place in the shape, whatever the strides."""
    rng = np.random.default_rng(5)
    m = lambda *s: make(rng, *s, dtype=BF16, grad=True)  # noqa: E731
    res = None
    if how == "heads":
        x = m(2, 3, 17, D).transpose(1, 2)
        res = m(2, 17, 3, D)
    elif how == "slice":
        x = m(4, 6, 200)[..., 64:64 + D]
    elif how == "offset":
        x = m(30 * D + 1)[1:].view(30, D)
    elif how == "odd_slice":
        x, res = m(4, 6, 201)[..., 3:3 + D], m(4, 6, 200)[..., 5:5 + D]
    elif how == "expanded":
        x, res = m(1, 5, D).expand(3, 5, D), m(3, 1, D).expand(3, 5, D)
    elif how == "last_axis":
        x, res = m(D, 11).t(), m(11, D)
    elif how == "six_axes":
        x = m(2, 3, 2, 5, 3, D).permute(4, 2, 0, 3, 1, 5)
    else:
        x, res = m(2, 17, 3, D), m(2, 3, 17, D).transpose(1, 2)
    g = case(x, res)
    if how == "heads":   # the gradient in the heads' own layout
        assert g.transpose(1, 2).is_contiguous()
    case(x, res, dy=torch.ones((), dtype=BF16, device="cuda").expand(x.shape))


def test_strides_below_zero_in_the_c_interface():
    n, D = 300, 64
    x = make(np.random.default_rng(6), n, D, dtype=BF16)
    back, y = x.flip(0).contiguous(), torch.empty_like(x)
    axes = lambda *s: (ctypes.c_longlong * len(s))(*s)  # noqa: E731
    code = _lib.dtype_code(BF16)
    assert _lib.load().mlstm_b200_dropout(back.data_ptr() + (n - 1) * D * 2, axes(0, 0, -D), None, None, y.data_ptr(), axes(0, 0, D), axes(1, 1, n, D),
                                          0.3, SEED, None, OFFSET, code, code, torch.cuda.current_stream().cuda_stream) == 0
    assert torch.equal(y, mk.dropout__b200(x, 0.3, SEED, OFFSET))


def test_seed_on_the_device():
    rng = np.random.default_rng(3)
    x, r = make(rng, 5, 100, dtype=BF16, grad=True), make(rng, 5, 100, dtype=BF16, grad=True)
    seed = torch.tensor([SEED], device="cuda")
    case(x, r, seed=seed)
    case(x, None, seed=seed.view(()))
    assert torch.equal(mk.dropout__b200(x, 0.3, seed, 3, r), mk.dropout__b200(x, 0.3, SEED, 3, r))
    a = [mk.dropout__b200(x, 0.3, s, o) != 0 for s, o in ((1, 0), (2, 0), (1, 1), (1 << 32, 0), (1, 1 << 32), (0, 0))]
    assert all(not torch.equal(p, q) for k, p in enumerate(a) for q in a[:k])
    y = mk.dropout__b200(x, 0.3, seed)
    seed.add_(1)
    with pytest.raises(RuntimeError, match="inplace"):   # another mask than the forward's
        y.sum().backward()


def test_share_and_independence():
    """Four million draws: shares of kept elements within six deviations of 1 - p, and of pairs of neighbours (in the row, the column, the
    next call) within six of (1 - p)^2."""
    x = torch.ones(2048, 2048, device="cuda")
    n = x.numel()
    for p in (0.1, 0.5):
        a, b = (mk.dropout__b200(x, p, 99, k) != 0 for k in (0, 1))
        q = 1 - p
        assert abs(a.double().mean().item() - q) < 6 * (q * p / n) ** 0.5
        for pair in (a & b, a[:, 1:] & a[:, :-1], a[1:] & a[:-1]):
            # neighbours share an element with the next pair: at most three times the variance of pairs apart
            assert abs(pair.double().mean().item() - q * q) < 6 * (3 * q * q * (1 - q * q) / pair.numel()) ** 0.5


def test_what_is_dropped_leaves_zeros():
    x = torch.full((1000,), float("nan"), device="cuda")
    x[::2] = float("inf")
    keep = torch.from_numpy(O.kept((1000,), 0.4, 5)).cuda()
    y = mk.dropout__b200(x, 0.4, 5)
    assert (y[~keep] == 0).all() and not torch.isfinite(y[keep]).any()
    assert torch.equal(mk.dropout__b200(x, 1.0, 5, residual=torch.ones_like(x)), torch.ones_like(x))


def test_gradients_of_one_of_the_two_and_none():
    rng = np.random.default_rng(3)
    x, r = make(rng, 5, 100, dtype=BF16, grad=True), make(rng, 5, 100, grad=True)
    case(x, r.detach())
    case(x.detach(), r)
    assert not mk.dropout__b200(x.detach(), 0.3, 1, residual=r.detach()).requires_grad
    y = mk.dropout__b200(x, 0.3, 1, residual=x)   # x in both places
    g, = torch.autograd.grad(y, x, torch.ones_like(y))
    keep = torch.from_numpy(O.kept(x.shape, 0.3, 1)).cuda()
    assert torch.equal(g, torch.where(keep, 1 + torch.tensor(1 / 0.7).bfloat16().cuda(), torch.ones((), dtype=BF16, device="cuda")))
    with pytest.raises(NotImplementedError, match="no second derivative"):
        torch.autograd.grad(mk.dropout__b200(x, 0.3, 1).float().sum(), x, create_graph=True)


def test_nothing():
    for shape in ((0,), (3, 0, 5), (0, 8)):
        x = torch.zeros(shape, device="cuda", requires_grad=True)
        y = mk.dropout__b200(x, 0.1, 1, residual=x)
        assert y.shape == shape
        assert torch.autograd.grad(y.sum(), x)[0].shape == shape


def test_offsets_past_32_bits():
    """More than 2^33 elements, whose counters need 33 bits: the last ones, and some in the middle, contiguous and strided."""
    n = (1 << 33) + (1 << 20) + 5
    x = torch.ones(n, dtype=BF16, device="cuda")
    y = mk.dropout__b200(x, 0.3, SEED, OFFSET)
    for at in (0, (1 << 31) - 1000, (1 << 32) - 1003, (1 << 33) + 77, n - 5000):
        assert np.array_equal(f64(y[at:at + 5000]) != 0, O.kept((min(5000, n - at),), 0.3, SEED, OFFSET, first=at)), at
    del y
    rows = x[:(1 << 33)].view(1 << 20, 1 << 13)[:, :4104 + 4000]
    y = mk.dropout__b200(rows, 0.3, SEED, OFFSET).view(-1)
    for at in ((1 << 32) - 1003, y.numel() - 5000):
        assert np.array_equal(f64(y[at:at + 5000]) != 0, O.kept((5000,), 0.3, SEED, OFFSET, first=at)), at


@pytest.mark.parametrize("n", [(1 << 31) - 5, (1 << 31) + (1 << 20) + 7])
def test_offsets_past_32_bits_of_any_alignment(n):
    x = torch.ones(n + 1, dtype=BF16, device="cuda")[1:]
    y = mk.dropout__b200(x, 0.3, SEED, OFFSET)
    for at in (0, (1 << 30) - 1003, n - 5000):
        assert np.array_equal(f64(y[at:at + 5000]) != 0, O.kept((5000,), 0.3, SEED, OFFSET, first=at)), at


@pytest.mark.parametrize("n", [1, 5, 31, 127, 128, 129, 1000, 1023, 1025, 4100])
@pytest.mark.parametrize("dtype,residual", PAIRS)
def test_lengths_off_the_boundary(n, dtype, residual):
    rng = np.random.default_rng(n)
    x = make(rng, n + 1, dtype=TDT[dtype])[1:].requires_grad_(True)
    case(x, None if residual is None else make(rng, n + 3, dtype=TDT[residual])[3:].requires_grad_(True))


def test_x_as_its_own_residual():
    x = make(np.random.default_rng(2), 33, 40, dtype=BF16, grad=True)
    y = mk.dropout__b200(x, 0.3, SEED, OFFSET, x)
    dy = make(np.random.default_rng(3), 33, 40, dtype=BF16)
    ref = O.dropout(f64(x), 0.3, SEED, OFFSET, f64(x), f64(dy))
    check(y, ref["y"], "y")
    g, = torch.autograd.grad(y, x, dy)
    alone = x.detach().clone().requires_grad_(True)
    d, = torch.autograd.grad(mk.dropout__b200(alone, 0.3, SEED, OFFSET), alone, dy)
    assert torch.equal(g, d + dy)


def test_captured_with_a_seed_that_counts():
    """A captured step with its seed on the GPU: each replay another mask, the same in forward and backward."""
    rng = np.random.default_rng(4)
    x, r = make(rng, 6, 500, dtype=BF16, grad=True), make(rng, 6, 500, grad=True)
    dy = torch.ones(6, 500, device="cuda")
    seed = torch.tensor([5], device="cuda")

    def run():
        y = mk.dropout__b200(x, 0.3, seed, 2, r)
        out = [y.detach(), *torch.autograd.grad(y, (x, r), dy)]
        seed.add_(1)
        return out
    run()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = run()
    for s in (5, 6, 1 << 40):
        seed.fill_(s)
        graph.replay()
        keep = torch.from_numpy(O.kept(x.shape, 0.3, s, 2)).cuda()
        assert torch.equal(captured[1] != 0, keep) and seed.item() == s + 1
        assert torch.equal(captured[0] != r, keep & (x != 0))
        assert torch.equal(captured[0], mk.dropout__b200(x, 0.3, s, 2, r))


def test_two_streams_and_another_thread_of_work():
    rng = np.random.default_rng(4)
    x, r = make(rng, 3000, 1024, dtype=BF16), make(rng, 3000, 1024)
    ref = mk.dropout__b200(x, 0.3, 1, 2, r)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for _ in range(5):
        for s in streams:
            with torch.cuda.stream(s):
                got.append(mk.dropout__b200(x, 0.3, 1, 2, r))
    torch.cuda.synchronize()
    assert all(torch.equal(g, ref) for g in got)


def test_compiled():
    rng = np.random.default_rng(4)
    x, r = make(rng, 2, 3, 50, 64, dtype=BF16, grad=True), make(rng, 2, 50, 3, 64, grad=True)
    seed = torch.tensor([5], device="cuda")
    dy = make(rng, 2, 50, 3, 64)
    for s in (seed, 17):
        fn = lambda x, r: mk.dropout__b200(x.transpose(1, 2), 0.2, s, 3, r)  # noqa: E731
        y, z = fn(x, r), torch.compile(fn, fullgraph=True)(x, r)
        assert torch.equal(y, z)
        for a, b in zip(torch.autograd.grad(y, (x, r), dy), torch.autograd.grad(z, (x, r), dy)):
            assert torch.equal(a, b)
    test = ("test_schema", "test_faketensor")
    ops = torch.ops.mlstm_b200
    for res in (None, r.detach()):
        for s in (None, seed):
            torch.library.opcheck(ops.dropout, (x.detach().transpose(1, 2), res, s, 4, 0.2, 1), test_utils=test)
    torch.library.opcheck(ops.dropout_bw, (dy, seed, 0, 0.2, 1, BF16), test_utils=test)


# ---- as they are used -----------------------------------------------------------------------------------------------
def block(D, rng):
    """norm, projections, convolution, gated recurrence, projection, dropout onto the residual stream"""
    P = dict(nw=make(rng, D, grad=True), nb=make(rng, D, grad=True), cw=make(rng, D, 4, scale=0.5, grad=True),
             wg=make(rng, D, 3 * D, scale=0.1, dtype=BF16, grad=True), wo=make(rng, D, D, scale=0.1, dtype=BF16, grad=True),
             rate=(-torch.exp(make(rng, D, shift=-2.0))).requires_grad_(True))

    def prompt(x, seed, p, st=None):
        st = st or {}
        n = mk.layer_norm__b200(x.to(BF16), P["nw"], P["nb"])
        u, tail = mk.short_conv__b200(n, P["cw"], x_initial=st.get("tail"), return_last_states=True, activation="silu")
        f, i, z = (n @ P["wg"]).chunk(3, -1)
        y, h = mk.gated_scan__b200(u, f, i, z, P["rate"], st.get("h"), True, "variance")
        y = y @ P["wo"]
        return (mk.dropout__b200(y, p, seed, 1, x) if p else x + y), dict(tail=tail, h=h)

    def token(x, st):
        n = mk.layer_norm__b200(x.to(BF16), P["nw"], P["nb"])
        u, tail = mk.short_conv_step__b200(n, st["tail"], P["cw"], activation="silu")
        f, i, z = (n @ P["wg"]).chunk(3, -1)
        y, h = mk.gated_step__b200(u, f, st["h"], i, z, P["rate"], "variance")
        return x + y @ P["wo"], dict(tail=tail, h=h)
    return P, prompt, token


@pytest.mark.parametrize("S", [48, 700])
def test_a_block_of_them_prompt_then_tokens(S):
    """A training step gives all parameters their gradients; at inference a prompt in one call and then token by token gives what the whole
    sequence gives."""
    rng = np.random.default_rng(21)
    B, D = 2, 64
    P, prompt, token = block(D, rng)
    x = make(rng, B, S, D)
    seed = torch.tensor([1], device="cuda")
    out, _ = prompt(x, seed, 0.1)
    grads = torch.autograd.grad(out.square().mean(), list(P.values()))
    assert all(torch.isfinite(g).all() and (g != 0).any() for g in grads)
    assert out.dtype == F32
    with torch.no_grad():
        whole, end = prompt(x, seed, 0)
        got, st = prompt(x[:, :32], seed, 0)
        # products of another shape round to bf16 otherwise
        assert (got - whole[:, :32]).abs().max() < 3e-2 * whole.abs().max()
        for t in range(32, 48):
            y, st = token(x[:, t], st)
            assert (y - whole[:, t]).abs().max() < 3e-2 * whole.abs().max()
        if S == 48:
            assert (st["h"] - end["h"]).abs().max() < 2e-2 * end["h"].abs().max()


def test_a_block_in_a_captured_step():
    """Forward and backward of the block in one graph, its seed counted up by the graph: the same as eager steps with these seeds."""
    rng = np.random.default_rng(22)
    P, prompt, _ = block(64, rng)
    x = make(rng, 2, 130, 64)
    seed = torch.tensor([7], device="cuda")

    def step():
        out, _ = prompt(x, seed, 0.2)
        g = torch.autograd.grad(out.square().mean(), list(P.values()))
        seed.add_(1)
        return [out.detach(), *g]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        eager = [step() for _ in range(3)]   # seeds 7, 8, 9
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    seed.fill_(8)
    for want in eager[1:]:
        graph.replay()
        for a, b in zip(want, captured):
            # (library products may be chosen otherwise in a capture)
            assert (a.float() - b.float()).abs().max() <= 2.0 ** -6 * a.float().abs().max()
