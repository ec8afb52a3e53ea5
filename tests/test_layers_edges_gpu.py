"""The operators around a recurrence on the GPU where values grow, vanish or end a type's range, against the oracle in float64."""

import numpy as np
import pytest
import torch

import mlstm_kernels_b200 as mk
from mlstm_kernels_b200 import _lib
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


# Logistic functions of f32 inputs.  In units of 2^-24 of e^x: 2^x off by 2^-22 (4), the exponent's rounding put back (1 for the
# factor, 1 for the product); of 1 / (1 + e): a sum (1), a reciprocal (2); a product (1): 10.  Twelve leave room for second orders.
UNITS = 12 * 2.0 ** -24


def sigmoid64(v):
    return 1 / (1 + np.exp(-v))


def relative(got, value, tol):
    g = f64(got)
    assert (np.abs(g - value) <= tol).all(), (np.abs(g - value) / np.maximum(tol, 1e-300)).max()


@pytest.mark.parametrize("D", [64, 63])   # four channels to a thread, and one
@pytest.mark.parametrize("S", [1, 70])
def test_silu_of_f32_keeps_its_digits(D, S):
    """u sigmoid(u) down to u = -80, where an argument rounded to f32 alone would cost 57 units."""
    rng = np.random.default_rng(S)
    x = torch.from_numpy(rng.uniform(-80, 20, (3, S, D))).float().cuda().requires_grad_(True)
    w = torch.zeros(D, 4, device="cuda")
    w[:, 3] = 1
    y = mk.short_conv__b200(x, w, activation="silu")
    u = f64(x)
    s = sigmoid64(u)
    relative(y, u * s, np.abs(u * s) * UNITS)
    g, = torch.autograd.grad(y, x, torch.ones_like(y))
    # s (1 + u (1 - s)): 1 - s is off by s's units and one of its own, so that the bracket is off by at most twice these of 1 + |u|
    relative(g, s * (1 + u * (1 - s)), s * (1 + np.abs(u)) * 3 * UNITS)
    one, _ = mk.short_conv_step__b200(x[:, -1].detach(), torch.zeros(3, 3, D, device="cuda"), w, activation="silu")
    assert torch.equal(one, y[:, -1])
    for v, want in ((float("inf"), float("inf")), (-200.0, 0.0), (200.0, 200.0)):
        assert (mk.short_conv__b200(torch.full((1, 1, D), v, device="cuda"), w[:, 2:], activation="silu") == want).all()


@pytest.mark.parametrize("D", [64, 63])
@pytest.mark.parametrize("S", [1, 70, 600])
def test_gate_of_f32_keeps_its_digits(D, S):
    rng = np.random.default_rng(S)
    z = torch.from_numpy(rng.uniform(-80, 20, (1, S, D))).float().cuda().requires_grad_(True)
    x = torch.ones(1, S, D, device="cuda").requires_grad_(True)
    nil, a, skip = torch.zeros(1, S, 4, device="cuda"), torch.zeros(D, 4, device="cuda"), torch.ones(D, device="cuda")
    y = mk.ssm_scan__b200(x, x.detach(), a, nil, nil, skip, z)
    v = f64(z)
    s = sigmoid64(v)
    relative(y, v * s, np.abs(v * s) * UNITS)
    gz, gx = torch.autograd.grad(y, (z, x), torch.ones_like(y))
    relative(gz, s * (1 + v * (1 - s)), s * (1 + np.abs(v)) * 3 * UNITS)
    relative(gx, v * s, np.abs(v * s) * UNITS)
    one, _ = mk.ssm_step__b200(x[:, -1].detach(), x[:, -1].detach(), a, nil[:, -1], nil[:, -1], torch.zeros(1, D, 4, device="cuda"), skip, z[:, -1].detach())
    relative(one, (v * s)[:, -1], np.abs(v * s)[:, -1] * UNITS)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("D", [64, 63])
def test_steps_keep_their_digits(D, dtype):
    """softplus down to -80 as the f32 state of one token shows it: e^x (6 units), its half logarithm s = e / (2 + e) (sum 1, reciprocal 2,
    product 1), the polynomial (2^-26 and four roundings: 5) and its product (1), and step * x and its product with b (2): 18.  A dt of 16 bits, itself off by 2^12 times that, leaves the rounding of
    the exponent in: 2 |dt| more."""
    rng = np.random.default_rng(D)
    T = TDT[dtype]
    dt = torch.from_numpy(rng.uniform(-80, 20, (40, 1, D))).to(T).cuda().requires_grad_(True)
    x, one = torch.ones(40, 1, D, dtype=T, device="cuda"), torch.ones(40, 1, 4, dtype=T, device="cuda")
    a = torch.zeros(D, 4, device="cuda")
    _, h = mk.ssm_scan__b200(x, dt, a, one, one, softplus=True, return_last_states=True)
    v = f64(dt)[:, 0, :, None] + np.zeros(4)
    step = np.logaddexp(v, 0)
    tol = step * (18 + (0 if dtype == "f32" else 2 * np.abs(v))) * 2.0 ** -24
    relative(h, step, tol)
    _, h = mk.ssm_step__b200(x[:, 0], dt[:, 0].detach(), a, one[:, 0], one[:, 0], torch.zeros(40, D, 4, device="cuda"), softplus=True)
    relative(h, step, tol)
    if dtype == "f32":   # the derivative, the logistic function: 12 units as above, and four products and sums
        _, h = mk.ssm_scan__b200(x, dt, a, one, one, softplus=True, return_last_states=True)
        g, = torch.autograd.grad(h, dt, torch.ones_like(h))
        s = 4 * sigmoid64(f64(dt))
        relative(g, s, s * 16 * 2.0 ** -24)


def test_nothing_in_and_nothing_out():
    """Batches and sequences of length zero: the shapes, and the state that goes through."""
    z = lambda *s: torch.zeros(*s, device="cuda")  # noqa: E731
    for B, S in ((2, 0), (0, 3), (0, 0)):
        x, bc, h0 = z(B, S, 8), z(B, S, 16), torch.ones(B, 8, 16, device="cuda")
        y, h = mk.ssm_scan__b200(x, x, z(8, 16), bc, bc, h_initial=h0, return_last_states=True)
        assert y.shape == x.shape and h.shape == h0.shape and torch.equal(h, h0)
        assert h.numel() == 0 or h.data_ptr() != h0.data_ptr()
        y, last = mk.short_conv__b200(x, z(8, 4), x_initial=torch.ones(B, 3, 8, device="cuda"), return_last_states=True)
        assert y.shape == x.shape and last.shape == (B, 3, 8) and (last == 1).all()
        assert mk.layer_norm__b200(x).shape == x.shape


@pytest.mark.parametrize("B,S,D,N,G,dtype", [(3, 700, 512, 128, 1, "bf16"), (2, 500, 1040, 100, 8, "f32"), (5, 333, 512, 128, 4, "bf16")])
def test_sums_over_channels_in_several_launches(B, S, D, N, G, dtype):
    """So many states and channels that the sums of db and dc do not find room for all segments at once: as one sequence after the other,
    and the sums over sequences (da, dskip, ddt_bias) as their sums."""
    lib = _lib.load()
    parts = G * -(-(D // G) // 8)   # CTAs' sums to a token, 2 KB each
    assert parts * B * S * 1024 > max(64 << 20, 2 * lib.mlstm_b200_ssm_checkpoint_bytes(B, S, D, N))
    rng = np.random.default_rng(S)
    T = TDT[dtype]
    m = lambda *s: make(rng, *s, dtype=T)  # noqa: E731
    t = dict(x=m(B, S, D), dt=m(B, S, D), a=-torch.exp(make(rng, D, N)), b=m(B, S, G, N), c=m(B, S, G, N), skip=make(rng, D), z=m(B, S, D),
             dt_bias=make(rng, D, shift=-2.0), h_initial=make(rng, B, D, N))
    dy = m(B, S, D)
    tok = ("x", "dt", "b", "c", "z", "h_initial")

    def grads(t, dy):
        t = {n: v.detach().requires_grad_(True) for n, v in t.items()}
        return dict(zip(t, torch.autograd.grad(mk.ssm_scan__b200(**t, softplus=True), list(t.values()), dy)))
    whole = grads(t, dy)
    alone = [grads({n: v[i:i + 1] if n in tok else v for n, v in t.items()}, dy[i:i + 1]) for i in range(B)]
    for n, g in whole.items():
        other = torch.cat([a[n] for a in alone]) if n in tok else sum(a[n].double() for a in alone)
        # other segments: f32 roundings of up to S steps' decays, at most a step of a 16-bit result
        far = (g.double() - other.double()).norm() / other.double().norm()
        assert far <= (S * 2.0 ** -24 if g.dtype == torch.float32 else 2.0 ** -9), (n, far.item())
    # a few channels of one sequence against the oracle
    i, at = B - 1, slice(0, 12)
    if G == 1:
        few = {n: (v[i:i + 1] if n in tok else v) for n, v in t.items()}
        few = {n: v if n in ("b", "c") else v[at] if n in ("a", "skip", "dt_bias") else v[:, at] if n == "h_initial" else v[..., at] for n, v in few.items()}
        ref = O.ssm_scan(**{n: f64(v) for n, v in few.items()}, softplus=True, dy=f64(dy[i:i + 1, :, at]), summed=S)
        check(whole["x"][i:i + 1, :, at], ref["dx"], "dx")
        check(whole["dt"][i:i + 1, :, at], ref["ddt"], "ddt")
