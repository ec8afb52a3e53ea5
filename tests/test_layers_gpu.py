"""The operators around a recurrence on the GPU, against the oracle in float64."""

import numpy as np
import pytest
import torch

import mlstm_kernels_b200 as mk
from oracle import layers_oracle as O
from util_layers import TDT, check, f64, make

pytestmark = pytest.mark.gpu

DTYPES = ["f32", "bf16", "f16"]


# ---- layer norm -----------------------------------------------------------------------------------------------------
def norm_case(x, w, b, dy, eps=1e-5):
    """x as the call gets it; dy in y's shape"""
    r = O.layer_norm(f64(x), f64(w), f64(b), eps, dy=f64(dy))
    y = mk.layer_norm__b200(x, w, b, eps)
    assert y.dtype == x.dtype and y.is_contiguous()
    check(y, r["y"], "y")
    leaves = [t for t in (x, w, b) if t is not None]
    grads = dict(zip([n for n, t in (("dx", x), ("dweight", w), ("dbias", b)) if t is not None], torch.autograd.grad(y, leaves, dy)))
    for n, g in grads.items():
        check(g, r[n], n)
    with torch.no_grad():
        assert torch.equal(mk.layer_norm__b200(x, w, b, eps), y)
    return grads


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D", [1, 2, 7, 8, 31, 64, 248, 256, 257, 264, 512, 520, 1000, 1001, 1024, 1032, 1500, 1536, 2048, 2056, 2500, 2900, 3500, 4096, 4104, 8192, 8200,
                               16383, 16384])
def test_layer_norm_widths(D, dtype):
    rng = np.random.default_rng(D)
    rows = 37 if D < 4096 else 5
    x = make(rng, rows, D, dtype=TDT[dtype], shift=0.5, grad=True)
    pdt = torch.float32 if D % 3 else TDT[dtype]
    norm_case(x, make(rng, D, dtype=pdt, grad=True), make(rng, D, dtype=pdt, grad=True), make(rng, rows, D, dtype=TDT[dtype]))


@pytest.mark.parametrize("rows", [1, 2, 7, 8, 9, 2000, 6001])
@pytest.mark.parametrize("weights", ["both", "weight", "bias", "none"])
def test_layer_norm_rows_and_weights(rows, weights):
    rng = np.random.default_rng(rows)
    D = 96
    x = make(rng, rows, D, grad=True)
    w = make(rng, D, grad=True) if weights in ("both", "weight") else None
    b = make(rng, D, grad=True) if weights in ("both", "bias") else None
    norm_case(x, w, b, make(rng, rows, D))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("B,NH,S,D", [(2, 4, 9, 256), (1, 3, 1, 64), (3, 1, 5, 40), (2, 5, 33, 129), (1, 2, 3, 1024), (1, 700, 3, 8)])
def test_layer_norm_of_heads_in_place(B, NH, S, D, dtype):
    """The output of a recurrence, (B, NH, S, D), as (B, S, NH, D): read through its strides, and the gradient in its layout."""
    rng = np.random.default_rng(S)
    h = make(rng, B, NH, S, D, dtype=TDT[dtype], shift=-0.3, grad=True)
    x = h.transpose(1, 2)
    g = norm_case(x, make(rng, NH, D, grad=True), make(rng, NH, D, grad=True), make(rng, B, S, NH, D, dtype=TDT[dtype]))
    assert g["dx"].transpose(1, 2).is_contiguous()


@pytest.mark.parametrize("how", ["slice", "offset", "expanded", "one_dim", "five_dims", "last_axis"])
def test_layer_norm_strides(how):
    rng = np.random.default_rng(5)
    D = 72
    w, b = make(rng, D, grad=True), make(rng, D, grad=True)
    dt = torch.bfloat16
    if how == "slice":         # the middle of wider rows
        x = make(rng, 4, 6, 200, dtype=dt, grad=True)[..., 64:64 + D]
    elif how == "offset":      # rows that no wide access fits
        x = make(rng, 30 * D + 1, dtype=dt, grad=True)[1:].view(30, D)
    elif how == "expanded":
        x = make(rng, 1, 5, D, dtype=dt, grad=True).expand(3, 5, D)
    elif how == "one_dim":
        x = make(rng, D, dtype=dt, grad=True)
    elif how == "five_dims":
        x = make(rng, 2, 3, 4, 5, D, dtype=dt, grad=True).permute(2, 0, 3, 1, 4)
    else:
        x = make(rng, D, 11, dtype=dt, grad=True).t()
    norm_case(x, w, b, make(rng, *x.shape, dtype=dt))
    # a gradient that is one number for all, without memory of its own
    y = mk.layer_norm__b200(x, w, b, 1e-5)
    r = O.layer_norm(f64(x), f64(w), f64(b), 1e-5, dy=np.ones(x.shape))
    for n, g in zip(("dx", "dweight", "dbias"), torch.autograd.grad(y.sum(), (x, w, b))):
        check(g, r[n], n)


@pytest.mark.parametrize("shape", [(3, 40), (1, 40), (2, 1, 40), (5, 5)])
def test_layer_norm_of_heads_alone(shape):
    """(NH, D) itself, one head, and as many heads as elements."""
    rng = np.random.default_rng(9)
    norm_case(make(rng, *shape, grad=True), make(rng, *shape[-2:], grad=True), make(rng, *shape[-2:], grad=True), make(rng, *shape))


def test_layer_norm_constant_rows_and_far_means():
    x = torch.full((3, 64), 7.0, device="cuda")
    assert (mk.layer_norm__b200(x) == 0).all()
    rng = np.random.default_rng(8)
    y = mk.layer_norm__b200(make(rng, 5, 300, shift=1000.0))
    assert torch.isfinite(y).all() and (y.mean(-1).abs() < 1e-3).all() and (y.std(-1) - 1).abs().max() < 1e-2
    x = make(rng, 4, 64)
    x[1, 3] = float("nan")
    y = mk.layer_norm__b200(x)
    assert y[1].isnan().all() and torch.isfinite(y[[0, 2, 3]]).all()


# ---- short convolution ----------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("W", [2, 3, 4])
@pytest.mark.parametrize("B,S,D", [(1, 1, 8), (2, 2, 5), (2, 3, 64), (3, 15, 1), (1, 16, 96), (2, 17, 260), (2, 31, 12), (1, 33, 1001), (2, 100, 72),
                                   (5, 64, 2)])
def test_short_conv(B, S, D, W, dtype):
    rng = np.random.default_rng(S * W)
    T = TDT[dtype]
    silu, init, bias = S % 2 == 0 or W == 4, W != 2, D != 64
    pdt = torch.float32 if W == 3 else T
    x, w = make(rng, B, S, D, dtype=T, grad=True), make(rng, D, W, dtype=pdt, grad=True)
    b = make(rng, D, dtype=pdt, grad=True) if bias else None
    x0 = make(rng, B, W - 1, D, dtype=T, grad=True) if init else None
    dy, dl = make(rng, B, S, D, dtype=T), make(rng, B, W - 1, D, dtype=T)
    r = O.short_conv(f64(x), f64(w), f64(b), f64(x0), silu, dy=f64(dy), dlast=f64(dl))
    y, last = mk.short_conv__b200(x, w, b, x0, return_last_states=True, activation="silu" if silu else None)
    check(y, r["y"], "y")
    assert np.array_equal(f64(last), r["last"][0])
    names = [n for n, t in (("dx", x), ("dweight", w), ("dbias", b), ("dx_initial", x0)) if t is not None]
    leaves = [t for t in (x, w, b, x0) if t is not None]
    for n, g in zip(names, torch.autograd.grad((y, last), leaves, (dy, dl))):
        check(g, r[n], n)
    # only y, and nothing of the tokens before; only the last tokens
    y = mk.short_conv__b200(x, w, b, x0, activation="silu" if silu else None)
    r = O.short_conv(f64(x), f64(w), f64(b), f64(x0), silu, dy=f64(dy))
    for n, g in zip(names, torch.autograd.grad(y, leaves, dy)):
        check(g, r[n], n)
    _, last = mk.short_conv__b200(x, w, b, x0, return_last_states=True)
    g = torch.autograd.grad(last, leaves, dl, allow_unused=True)
    assert np.array_equal(f64(g[0])[:, max(0, S - (W - 1)):], f64(dl)[:, max(0, W - 1 - S):])
    assert (g[0][:, :max(0, S - (W - 1))] == 0).all() and (g[1] == 0).all()


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_short_conv_of_a_slice_and_many_tokens(dtype):
    """x and dy as parts of wider rows, at an offset that no wide access fits too; more runs than one CTA takes."""
    rng = np.random.default_rng(11)
    T = TDT[dtype]
    B, S, D, W = 3, 700, 40, 4
    for off in (8, 3):
        wide = make(rng, B, S, 128, dtype=T, grad=True)
        x = wide[..., off:off + D]
        w, b = make(rng, D, W, grad=True), make(rng, D, grad=True)
        dy = make(rng, S, B, 64, dtype=T)[..., off:off + D].transpose(0, 1)
        r = O.short_conv(f64(x), f64(w), f64(b), None, True, dy=f64(dy))
        y = mk.short_conv__b200(x, w, b, activation="silu")
        check(y, r["y"], "y")
        for n, g in zip(("dx", "dweight", "dbias"), torch.autograd.grad(y, (x, w, b), dy)):
            check(g, r[n], n)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("B,D,W", [(1, 8, 2), (3, 65, 4), (17, 1024, 3)])
def test_short_conv_tokens_one_by_one(B, D, W, dtype):
    """The step is the convolution: token by token from the last tokens of a prompt, bit for bit; in place too."""
    rng = np.random.default_rng(D)
    T = TDT[dtype]
    S = 9
    x, w, b = make(rng, B, S, D, dtype=T), make(rng, D, W, dtype=T), make(rng, D, dtype=T)
    whole, end = mk.short_conv__b200(x, w, b, return_last_states=True, activation="silu")
    y, state = mk.short_conv__b200(x[:, :4], w, b, return_last_states=True, activation="silu")
    kept = state.clone()
    for t in range(4, S):
        y, new = mk.short_conv_step__b200(x[:, t], state, w, b, activation="silu")
        assert torch.equal(y, whole[:, t])
        if t == 4:
            assert torch.equal(state, kept)
            state = new
        else:
            y2, same = mk.short_conv_step__b200(x[:, t], state, w, b, activation="silu", state_new=state)
            assert same is state and torch.equal(y2, y) and torch.equal(state, new)
    assert torch.equal(state, end)


def test_a_steps_buffer_lies_apart_from_what_it_reads():
    """The new state may be written over the whole old one and over nothing else, and autograd knows of the write."""
    rng = np.random.default_rng(8)
    B, D, W, N = 3, 16, 4, 8
    f = lambda *shape: make(rng, *shape, dtype=torch.float32)
    pool = f(2 * B * (W - 1) * D)
    state, shifted = (pool[at : at + B * (W - 1) * D].view(B, W - 1, D) for at in (0, D))
    x, w = f(B, D), f(D, W)
    conv = lambda **o: mk.short_conv_step__b200(**{**dict(x=x, state=state, weight=w), **o})
    before = pool.clone()
    for o in (dict(state_new=shifted), dict(state=shifted, state_new=state), dict(state_new=state, x=pool[D : D + B * D].view(B, D)),
              dict(state_new=shifted, state=f(B, W - 1, D), weight=pool[: D * W].view(D, W))):
        with pytest.raises(ValueError, match="state_new overlaps"):
            conv(**o)
    hp = f(2 * B * D * N)
    h, h_shifted = (hp[at : at + B * D * N].view(B, D, N) for at in (0, N))
    args = dict(x=x, dt=f(B, D), a=f(D, N), b=f(B, N), c=f(B, N), h=h)
    h_before = hp.clone()
    for o in (dict(h_new=h_shifted), dict(h=h_shifted, h_new=h), dict(h_new=h, x=hp[: B * D].view(B, D)), dict(h_new=h, a=hp[D : D + D * N].view(D, N))):
        with pytest.raises(ValueError, match="h_new overlaps"):
            mk.ssm_step__b200(**{**args, **o})
    assert torch.equal(pool, before) and torch.equal(hp, h_before)
    # the rest of a pool, and an inference tensor, are as good as any
    y, new = conv()
    assert torch.equal(conv(state_new=pool[B * (W - 1) * D :].view(B, W - 1, D))[1], new) and torch.equal(state, before[: state.numel()].view_as(state))
    with torch.inference_mode():
        assert torch.equal(conv(state_new=torch.empty_like(state))[1], new)
    # a graph that kept the old state
    wl = w.clone().requires_grad_()
    out = mk.short_conv__b200(f(B, 5, D), wl, x_initial=state)
    conv(state_new=state)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        out.sum().backward()
    hl = h.clone().requires_grad_()
    out = (hl * h).sum()
    mk.ssm_step__b200(**args, h_new=h)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        out.backward()


# ---- selective state space scan -------------------------------------------------------------------------------------
def ssm_inputs(seed, B, S, D, N, G, dtype, gate=True, init=True, softplus=True, skip=True, grad=True):
    rng = np.random.default_rng(seed)
    T = TDT[dtype]
    m = lambda *s, **k: make(rng, *s, grad=grad, **k)  # noqa: E731
    bc = (B, S, N) if G == 0 else (B, S, G, N)
    t = dict(x=m(B, S, D, dtype=T), dt=m(B, S, D, dtype=T) if softplus else m(B, S, D, dtype=T, scale=0.02, shift=0.1))
    t["a"] = -torch.exp(make(rng, D, N)).detach()
    if grad:
        t["a"].requires_grad_(True)
    t["b"], t["c"] = m(*bc, dtype=T), m(*bc, dtype=T)
    if skip:
        t["skip"] = m(D)
    if gate:
        t["z"] = m(B, S, D, dtype=T)
    if softplus:
        t["dt_bias"] = m(D, shift=-2.0)
    if init:
        t["h_initial"] = m(B, D, N)
    return t


def ssm_case(t, softplus, seed=0, last=True, dy=None, summed=0):
    rng = np.random.default_rng(1000 + seed)
    T = t["x"].dtype
    B, S, D = t["x"].shape
    dy = make(rng, B, S, D, dtype=T) if dy is None else dy
    dh = make(rng, B, D, t["a"].shape[1]) if last else None
    ref = O.ssm_scan(**{n: f64(v) for n, v in t.items()}, softplus=softplus, dy=f64(dy), dh_last=f64(dh), summed=summed)
    y, h = mk.ssm_scan__b200(**t, softplus=softplus, return_last_states=True)
    assert y.dtype == T and h.dtype == torch.float32
    check(y, ref["y"], "y")
    check(h, ref["h_last"], "h_last")
    outs, ups = ((y, h), (dy, dh)) if last else ((y,), (dy,))
    for n, g in zip(t, torch.autograd.grad(outs, list(t.values()), ups)):
        assert g.dtype == t[n].dtype
        check(g, ref["d" + n], "d" + n)
    with torch.no_grad():
        y2 = mk.ssm_scan__b200(**t, softplus=softplus)
        assert torch.equal(y, y2)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("N", [1, 2, 4, 5, 8, 9, 16, 17, 32, 33, 64, 65, 128])
def test_ssm_state_sizes(N, dtype):
    ssm_case(ssm_inputs(N, 2, 37, 36, N, 0, dtype), True)


@pytest.mark.parametrize("S", [1, 2, 15, 16, 17, 31, 32, 33, 100])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_ssm_lengths(S, dtype):
    ssm_case(ssm_inputs(S, 3, S, 68, 16, 0, dtype), True)


@pytest.mark.parametrize("D,G", [(1, 0), (3, 1), (64, 2), (65, 5), (66, 3), (130, 2), (256, 4), (260, 0)])
@pytest.mark.parametrize("dtype", ["f32", "f16"])
def test_ssm_channels_and_groups(D, G, dtype):
    ssm_case(ssm_inputs(D, 2, 21, D, 12, G, dtype), True)


@pytest.mark.parametrize("gate", [False, True])
@pytest.mark.parametrize("init", [False, True])
@pytest.mark.parametrize("softplus,skip,last", [(True, False, False), (False, True, True), (False, False, False)])
def test_ssm_options(gate, init, softplus, skip, last):
    ssm_case(ssm_inputs(7, 2, 40, 48, 16, 1, "bf16", gate, init, softplus, skip), softplus, last=last)


@pytest.mark.parametrize("B,S,D,N,G", [(1, 1000, 64, 16, 0), (2, 777, 24, 16, 2), (1, 600, 8, 3, 0), (1, 500, 40, 64, 0), (1, 321, 12, 128, 1)])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_ssm_long_sequences_in_segments(B, S, D, N, G, dtype):
    """Few channels and many tokens: the sequence is cut, forward and backward."""
    from mlstm_kernels_b200 import _lib
    assert _lib.load().mlstm_b200_ssm_workspace_bytes(B, S, D, N, max(G, 1), 0) > 0
    ssm_case(ssm_inputs(S, B, S, D, N, G, dtype), True, summed=S)


def test_ssm_many_channels():
    """More tiles of channels than CTAs that write sums: each CTA takes several, one after the other."""
    ssm_case(ssm_inputs(12, 1, 20, 70 * 8 - 4, 128, 0, "f32"), True)
    ssm_case(ssm_inputs(13, 2, 33, 2 * 131 * 8, 100, 2, "bf16"), True)


def test_ssm_strides():
    """Operands as parts of wider rows, at offsets that no wide access fits too; a gradient without memory of its own."""
    rng = np.random.default_rng(3)
    B, S, D, N = 2, 50, 40, 16
    t = ssm_inputs(9, B, S, D, N, 0, "bf16")
    for off in (0, 8, 5):
        wide = make(rng, S, B, 160, dtype=torch.bfloat16, grad=True).transpose(0, 1)
        rows = make(rng, B, S, 100, dtype=torch.bfloat16, grad=True)
        t.update(x=wide[..., off:off + D], z=wide[..., off + D:off + 2 * D], b=rows[..., off:off + N], c=rows[..., 40:40 + N])
        ssm_case(t, True)
    ssm_case(t, True, dy=torch.ones((), dtype=torch.bfloat16, device="cuda").expand(B, S, D))
    t["b"] = make(rng, B, N, S, dtype=torch.bfloat16, grad=True).transpose(1, 2)   # the last axis apart
    ssm_case(t, True)


def test_ssm_only_the_last_state_and_only_some_gradients():
    t = ssm_inputs(14, 2, 45, 40, 16, 2, "bf16")
    dh = make(np.random.default_rng(2), 2, 40, 16)
    ref = O.ssm_scan(**{n: f64(v) for n, v in t.items()}, softplus=True, dy=np.zeros((2, 45, 40)), dh_last=f64(dh))
    _, h = mk.ssm_scan__b200(**t, softplus=True, return_last_states=True)
    for n, g in zip(t, torch.autograd.grad(h, list(t.values()), dh, allow_unused=True)):
        check(g, ref["d" + n], "d" + n)
    for n in ("a", "b", "h_initial"):   # one input alone wants a gradient
        only = {m: v.detach().requires_grad_(m == n) for m, v in t.items()}
        _, h = mk.ssm_scan__b200(**only, softplus=True, return_last_states=True)
        check(torch.autograd.grad(h, only[n], dh)[0], ref["d" + n], "d" + n)


def test_ssm_operands_without_memory_of_their_own():
    """b and c the same for all sequences, x the same for all tokens: strides of zero, and gradients summed by whoever expanded them."""
    rng = np.random.default_rng(6)
    B, S, D, N = 3, 40, 24, 16
    t = ssm_inputs(15, B, S, D, N, 0, "f32", grad=False)
    t["b"], t["c"] = (make(rng, 1, S, N).expand(B, S, N) for _ in range(2))
    t["x"] = make(rng, B, 1, D).expand(B, S, D)
    t = {n: v.requires_grad_(True) for n, v in t.items()}
    ssm_case(t, True)


def test_ssm_token_axis_of_any_stride():
    """One token, whose stride means nothing; and tokens too far apart for the kernels, which the call gathers first."""
    rng = np.random.default_rng(4)
    t = ssm_inputs(3, 2, 1, 24, 16, 0, "f32")
    t["x"] = make(rng, 2, 24).as_strided((2, 1, 24), (24, 1 << 40, 1)).requires_grad_(True)
    ssm_case(t, True)
    t = ssm_inputs(3, 1, 2, 8, 16, 0, "bf16")
    far = torch.zeros((1 << 29) + 8, dtype=torch.bfloat16, device="cuda")
    far[:8], far[-8:] = t["x"].detach()[0, 0], t["x"].detach()[0, 1]
    t["x"] = far.as_strided((1, 2, 8), (1 << 29, 1 << 29, 1)).requires_grad_(True)
    ssm_case(t, True)


def test_ssm_parameters_in_16_bits():
    t = ssm_inputs(5, 2, 20, 32, 16, 0, "bf16")
    for n in ("skip", "dt_bias", "h_initial"):
        t[n] = t[n].detach().bfloat16().requires_grad_(True)
    ssm_case(t, True)


def test_ssm_strong_and_no_decay():
    """Steps of zero leave the state as it was; rates of -2000 and steps of 30 forget it; neither makes anything but numbers."""
    t = ssm_inputs(6, 1, 40, 16, 16, 0, "f32", softplus=False)
    t["dt"] = torch.zeros(1, 40, 16, device="cuda", requires_grad=True)
    ssm_case(t, False)
    y, h = mk.ssm_scan__b200(**t, return_last_states=True)
    assert torch.equal(h, t["h_initial"])
    t["dt"] = torch.full((1, 40, 16), 30.0, device="cuda", requires_grad=True)
    t["a"] = torch.full((16, 16), -2000.0, device="cuda", requires_grad=True)
    ssm_case(t, False)


def test_ssm_nan_stays_in_its_channel():
    t = ssm_inputs(2, 2, 40, 32, 16, 0, "bf16", grad=False)
    t["x"][1, 5, 3] = float("nan")
    y, h = mk.ssm_scan__b200(**t, softplus=True, return_last_states=True)
    bad = torch.zeros_like(y, dtype=torch.bool)
    bad[1, 5:, 3] = True
    assert torch.equal(y.isnan(), bad)
    assert h[1, 3].isnan().all() and h.isnan().sum() == 16


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("B,D,N,G", [(1, 8, 16, 0), (3, 65, 5, 1), (2, 96, 64, 3), (5, 32, 128, 0), (2, 1000, 16, 0)])
def test_ssm_tokens_one_by_one(B, D, N, G, dtype):
    """A prompt, then single tokens from its last state."""
    S = 12
    t = ssm_inputs(D, B, S, D, N, G, dtype, grad=False)
    ref = O.ssm_scan(**{n: f64(v) for n, v in t.items()}, softplus=True)
    tok = ("x", "dt", "b", "c", "z")
    _, h = mk.ssm_scan__b200(**{n: v[:, :5] if n in tok else v for n, v in t.items()}, softplus=True, return_last_states=True)
    rest = {n: t[n] for n in ("a", "skip", "dt_bias")}
    for s in range(5, S):
        now = {n: t[n][:, s] for n in tok}
        old = h.clone()
        y, new = mk.ssm_step__b200(**now, **rest, h=h, softplus=True)
        assert torch.equal(h, old)
        check(y, (ref["y"][0][:, s], ref["y"][1][:, s]), "y")
        y2, same = mk.ssm_step__b200(**now, **rest, h=h, softplus=True, h_new=h)
        assert same is h and torch.equal(y, y2) and torch.equal(h, new)
    check(h, ref["h_last"], "h")


# ---- all of them ----------------------------------------------------------------------------------------------------
def calls(grad=True):
    rng = np.random.default_rng(1)
    t = ssm_inputs(4, 2, 300, 64, 16, 0, "bf16", grad=grad)
    x, w, b = make(rng, 2, 300, 64, dtype=torch.bfloat16, grad=grad), make(rng, 64, 4, grad=grad), make(rng, 64, grad=grad)
    return {"norm": (lambda: mk.layer_norm__b200(x, b, b), [x, b]),
            "conv": (lambda: mk.short_conv__b200(x, w, b, activation="silu"), [x, w, b]),
            "ssm": (lambda: mk.ssm_scan__b200(**t, softplus=True), list(t.values()))}


@pytest.mark.parametrize("op", ["norm", "conv", "ssm"])
def test_same_bits_again_on_another_stream_and_from_a_graph(op):
    fn, leaves = calls()[op]
    dy = torch.ones(2, 300, 64, dtype=torch.bfloat16, device="cuda")

    def run():
        y = fn()
        return [y.detach(), *torch.autograd.grad(y, leaves, dy)]
    first = run()
    for a, b in zip(first, run()):
        assert torch.equal(a, b)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        second = run()
        for a, b in zip(first, second):
            assert torch.equal(a, b)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()   # (no eager graph of these leaves is alive: PyTorch would drag its stream into the capture)
    with torch.cuda.graph(graph):
        captured = run()
    with torch.cuda.graph(torch.cuda.CUDAGraph()):
        run()      # another capture, whose workspaces are its own
    for t in captured:
        t.zero_()
    graph.replay()
    for a, b in zip(first, captured):
        assert torch.equal(a, b)
    with torch.no_grad():
        leaves[0].mul_(0.5)   # a replay reads what the inputs hold then
    graph.replay()
    for a, b in zip(run(), captured):
        assert torch.equal(a, b)


def test_calls_on_two_streams_at_once():
    """The same inputs on two streams, neither waiting for the other: workspaces are each call's own."""
    jobs = {op: fn_leaves for op, fn_leaves in calls().items()}
    dy = torch.ones(2, 300, 64, dtype=torch.bfloat16, device="cuda")

    def run():
        out = []
        for fn, leaves in jobs.values():
            y = fn()
            out += [y.detach(), *torch.autograd.grad(y, leaves, dy)]
        return out
    alone = run()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(5):
        for s, g in zip(streams, got):
            with torch.cuda.stream(s):
                g[:] = run()
    torch.cuda.synchronize()
    for g in got:
        for a, b in zip(alone, g):
            assert torch.equal(a, b)


@pytest.mark.parametrize("op", ["norm", "conv", "ssm"])
def test_no_second_derivative(op):
    fn, leaves = calls()[op]
    with pytest.raises(NotImplementedError, match="no second derivative"):
        torch.autograd.grad(fn().float().sum(), leaves, create_graph=True)


def test_no_tokens():
    z = lambda *s, **k: torch.zeros(*s, device="cuda", **k)  # noqa: E731
    for B, S in ((2, 0), (0, 3)):
        x, w, b = z(B, S, 8, requires_grad=True), z(8, 4, requires_grad=True), z(8, requires_grad=True)
        x0 = torch.ones(B, 3, 8, device="cuda", requires_grad=True)
        y, last = mk.short_conv__b200(x, w, b, x0, return_last_states=True)
        assert y.shape == x.shape and torch.equal(last, x0)
        gx, gw, g0 = torch.autograd.grad(last.sum() + y.sum(), (x, w, x0))
        assert gx.shape == x.shape and (gw == 0).all() and (g0 == 1).all()
        assert (mk.short_conv__b200(x, w, b, return_last_states=True)[1] == 0).all()
        a, bc, h0 = z(8, 16, requires_grad=True), z(B, S, 16, requires_grad=True), torch.ones(B, 8, 16, device="cuda", requires_grad=True)
        y, h = mk.ssm_scan__b200(x, x, a, bc, bc, h_initial=h0, return_last_states=True)
        assert y.shape == x.shape and torch.equal(h, h0) and h.data_ptr() != h0.data_ptr() or h.numel() == 0
        ga, g0 = torch.autograd.grad(h.sum() + y.sum(), (a, h0))
        assert (ga == 0).all() and (g0 == 1).all()
        y = mk.layer_norm__b200(x, b, b)
        assert y.shape == x.shape
        assert (torch.autograd.grad(y.sum(), b)[0] == 0).all()
    y, s = mk.short_conv_step__b200(z(0, 8), z(0, 3, 8), z(8, 4))
    assert y.shape == (0, 8) and s.shape == (0, 3, 8)
    y, h = mk.ssm_step__b200(z(0, 8), z(0, 8), z(8, 4), z(0, 4), z(0, 4), z(0, 8, 4))
    assert y.shape == (0, 8) and h.shape == (0, 8, 4)


def test_gradient_of_the_kernels_is_that_of_the_formula_by_differences():
    """Along a random direction of all inputs: the oracle's value there and back against the kernels' gradients."""
    t = ssm_inputs(8, 2, 30, 12, 16, 0, "f32")
    rng = np.random.default_rng(2)
    w = rng.standard_normal((2, 30, 12))
    y = mk.ssm_scan__b200(**t, softplus=True)
    grads = torch.autograd.grad(y, list(t.values()), torch.from_numpy(w).float().cuda())
    w = f64(torch.from_numpy(w).float())
    dirs = {n: rng.standard_normal(v.shape) for n, v in t.items()}
    loss = lambda s: (O.ssm_scan(**{n: f64(v) + s * dirs[n] for n, v in t.items()}, softplus=True)["y"][0] * w).sum()  # noqa: E731
    d = (loss(1e-6) - loss(-1e-6)) / 2e-6
    terms = [(f64(g) * dirs[n]) for n, g in zip(t, grads)]
    size = sum(np.abs(v).sum() for v in terms)
    # of f32 gradients, each off by up to a few thousand units (decays over 30 tokens): 2^-12 of the absolute sum
    assert abs(d - sum(v.sum() for v in terms)) < size * 2.0 ** -12


@pytest.mark.parametrize("op", ["norm", "conv", "ssm"])
def test_compiled_without_graph_break(op):
    fn, leaves = calls()[op]
    dy = torch.ones(2, 300, 64, dtype=torch.bfloat16, device="cuda")
    y = fn()
    eager = [y, *torch.autograd.grad(y, leaves, dy)]
    y = torch.compile(fn, fullgraph=True)()
    for a, b in zip(eager, [y, *torch.autograd.grad(y, leaves, dy)]):
        assert torch.equal(a, b)


def test_compiled_for_any_length():
    t = ssm_inputs(4, 2, 50, 64, 16, 0, "bf16", grad=False)
    tok = ("x", "dt", "b", "c", "z")
    w = make(np.random.default_rng(1), 64, 4)

    def fn(t):
        u = mk.short_conv__b200(mk.layer_norm__b200(t["x"]), w, activation="silu")
        return mk.ssm_scan__b200(**{**t, "x": u}, softplus=True)
    compiled = torch.compile(fn, fullgraph=True, dynamic=True)
    for S in (50, 33, 41):
        cut = {n: v[:, :S].contiguous() if n in tok else v for n, v in t.items()}
        assert torch.equal(fn(cut), compiled(cut))


def test_steps_compile():
    rng = np.random.default_rng(1)
    x, s, w = make(rng, 3, 40), make(rng, 3, 3, 40), make(rng, 40, 4)
    a, b, h = -torch.exp(make(rng, 40, 16)), make(rng, 3, 16), make(rng, 3, 40, 16)

    def step(x, s, h):
        u, s = mk.short_conv_step__b200(x, s, w, activation="silu")
        y, h = mk.ssm_step__b200(u, x, a, b, b, h, softplus=True)
        return y, s, h
    for p, q in zip(step(x, s, h), torch.compile(step, fullgraph=True)(x, s, h)):
        assert torch.equal(p, q)


@pytest.mark.parametrize("op", ["norm", "conv", "ssm"])
def test_offsets_past_32_bits(op):
    """Tensors of more than 2^31 elements: the last sequence comes out as it does alone."""
    B, S, D = 521, 2048, 2048
    dt = torch.bfloat16
    rng = np.random.default_rng(3)
    x = torch.zeros(B, S, D, dtype=dt, device="cuda")
    assert x.numel() > 1 << 31
    x[-1] = make(rng, S, D, dtype=dt)
    w, par, bc = make(rng, D, 4), make(rng, D), make(rng, B, S, 16, dtype=dt)
    a = -torch.exp(make(rng, D, 16))
    fn = {"norm": lambda x, bc: mk.layer_norm__b200(x, par, par), "conv": lambda x, bc: mk.short_conv__b200(x, w, par, activation="silu"),
          "ssm": lambda x, bc: mk.ssm_scan__b200(x, x, a, bc, bc, par, None, par, True)}[op]

    def run(x, bc):
        x = x.requires_grad_(True)
        y = fn(x, bc)
        g, = torch.autograd.grad(y, x, x.detach())
        return y[-1].detach().clone(), g[-1].clone()
    for got, alone in zip(run(x, bc), run(x.detach()[-1:].clone(), bc[-1:])):
        # the scan may be cut into other segments, which moves f32 values by some units and so a few bf16 ones by a step
        assert torch.equal(got, alone) if op != "ssm" else (got.float() - alone.float()).abs().max() <= 2.0 ** -7 * alone.float().abs().max()


def test_a_layer_of_them_prompt_then_tokens():
    """As they are used: norm, convolution, scan and mLSTM side by side, norm of the heads; a prompt in one call and then token by
    token gives what the whole sequence gives, and all parameters get their gradients."""
    rng = np.random.default_rng(21)
    B, S, D, N, NH = 2, 48, 64, 16, 4
    T = torch.bfloat16
    P = dict(nw=make(rng, D, grad=True), nb=make(rng, D, grad=True), cw=make(rng, D, 4, scale=0.5, grad=True), wdt=make(rng, D, D, scale=0.1, dtype=T, grad=True),
             wb=make(rng, D, 2 * N, scale=0.1, dtype=T, grad=True), skip=make(rng, D, grad=True), dtb=make(rng, D, shift=-2.0, grad=True),
             hw=make(rng, NH, D // NH, grad=True), wg=make(rng, D, 2 * NH, scale=0.1, dtype=T, grad=True))
    a = -torch.exp(make(rng, D, N)).detach().requires_grad_(True)
    x = make(rng, B, S, D, dtype=T)

    def prompt(x, st=None):
        st = st or {}
        n = mk.layer_norm__b200(x, P["nw"], P["nb"])
        u, tail = mk.short_conv__b200(n, P["cw"], x_initial=st.get("tail"), return_last_states=True, activation="silu")
        b, c = (u @ P["wb"]).chunk(2, -1)
        y, h = mk.ssm_scan__b200(u, u @ P["wdt"], a, b, c, P["skip"], n, P["dtb"], True, st.get("h"), True)
        q = u.view(B, -1, NH, D // NH).transpose(1, 2)
        gi, gf = (u @ P["wg"]).transpose(1, 2).chunk(2, 1)
        m, cnm = mk.mlstm_chunkwise__b200_xl_chunk(q, q, q, gi, gf + 3, return_last_states=True)
        m = mk.layer_norm__b200(m.transpose(1, 2), P["hw"]).reshape(B, -1, D)
        return y + m, dict(tail=tail, h=h, cnm=cnm)

    def token(x, st):
        n = mk.layer_norm__b200(x, P["nw"], P["nb"])
        u, tail = mk.short_conv_step__b200(n, st["tail"], P["cw"], activation="silu")
        b, c = (u @ P["wb"]).chunk(2, -1)
        y, h = mk.ssm_step__b200(u, u @ P["wdt"], a, b, c, st["h"], P["skip"], n, P["dtb"], True)
        q = u.view(B, NH, D // NH)
        gi, gf = (u @ P["wg"]).unsqueeze(-1).chunk(2, 1)
        m, cnm = mk.mlstm_recurrent_step__b200(q, q, q, gi, gf + 3, *st["cnm"])
        return y + mk.layer_norm__b200(m, P["hw"]).reshape(B, D), dict(tail=tail, h=h, cnm=cnm)

    out, _ = prompt(x)
    grads = torch.autograd.grad(out.float().square().mean(), [*P.values(), a])
    assert all(torch.isfinite(g).all() and (g != 0).any() for g in grads)
    with torch.no_grad():
        whole, end = prompt(x)
        got, st = prompt(x[:, :32])
        assert torch.equal(got, whole[:, :32])
        for t in range(32, S):
            y, st = token(x[:, t], st)
            # the paths differ in roundings to bf16 of the mLSTM's operands and of products of a different shape
            assert (y.float() - whole[:, t].float()).abs().max() < 3e-2 * whole.float().abs().max()
        assert (st["h"] - end["h"]).abs().max() < 2e-2 * end["h"].abs().max()
