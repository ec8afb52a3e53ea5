"""The gated linear recurrence on the GPU, against the oracle in float64."""

import ctypes

import numpy as np
import pytest
import torch

import mlstm_kernels_b200 as mk
from mlstm_kernels_b200 import _lib
from oracle import gated_oracle as O
from util_layers import TDT, check, f64, make

pytestmark = pytest.mark.gpu

DTYPES = ["f32", "bf16", "f16"]
BF16 = torch.bfloat16
SCALES = [None, "convex", "variance"]
TOKENS = ("x", "f", "i", "z")


def inputs(seed, B, S, D, dtype, gates="iz", rate=True, init=True, shift=2.0, grad=True):
    rng = np.random.default_rng(seed)
    T = TDT[dtype]
    m = lambda *s, **k: make(rng, *s, grad=grad, **k)  # noqa: E731
    t = dict(x=m(B, S, D, dtype=T), f=m(B, S, D, dtype=T, shift=shift))
    for n in gates:
        t[n] = m(B, S, D, dtype=T)
    if rate:
        t["rate"] = -torch.exp(make(rng, D, shift=-2.0))
        t["rate"].requires_grad_(grad)
    if init:
        t["h_initial"] = m(B, D)
    return t


def case(t, scale, last=True, seed=0, dy=None):
    """y, the last state and all gradients against the oracle's; without gradients the same values."""
    rng = np.random.default_rng(1000 + seed)
    T = t["x"].dtype
    B, S, D = t["x"].shape
    dy = make(rng, B, S, D, dtype=T) if dy is None else dy
    dh = make(rng, B, D) if last else None
    ref = O.gated_scan(**{n: f64(v) for n, v in t.items()}, input_scale=scale, dy=f64(dy), dh_last=f64(dh))
    y, h = mk.gated_scan__b200(**t, input_scale=scale, return_last_states=True)
    assert y.dtype == T and h.dtype == torch.float32 and y.is_contiguous()
    check(y, ref["y"], "y")
    check(h, ref["h_last"], "h_last")
    outs, ups = ((y, h), (dy, dh)) if last else ((y,), (dy,))
    for n, g in zip(t, torch.autograd.grad(outs, list(t.values()), ups)):
        assert g.dtype == t[n].dtype
        check(g, ref["d" + n], "d" + n)
    with torch.no_grad():
        assert torch.equal(mk.gated_scan__b200(**t, input_scale=scale), y)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("S", [1, 2, 7, 8, 9, 15, 16, 17, 31, 33, 63, 64, 65, 127, 128, 129, 257, 600])
def test_lengths(S, dtype):
    case(inputs(S, 3, S, 72, dtype), "variance")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D", [1, 2, 3, 4, 5, 8, 16, 31, 32, 33, 62, 63, 64, 65, 66, 96, 126, 128, 130, 257, 1000, 1001, 2048])
def test_widths(D, dtype):
    case(inputs(D, 2, 37, D, dtype), "convex")


@pytest.mark.parametrize("scale", SCALES)
@pytest.mark.parametrize("gates", ["", "i", "z", "iz"])
@pytest.mark.parametrize("rate", [False, True])
@pytest.mark.parametrize("init,last", [(False, False), (True, True)])
def test_options(scale, gates, rate, init, last):
    for D in (40, 41):
        case(inputs(5, 2, 70, D, "bf16", gates, rate, init), scale, last)
    case(inputs(6, 2, 70, 40, "f32", gates, rate, init), scale, last)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("B,S,D", [(1, 5000, 64), (1, 3001, 1), (2, 2049, 40), (1, 4096, 200), (1, 2500, 33), (5, 1100, 96), (1, 1030, 2048), (1, 20000, 16)])
def test_few_channels_and_many_tokens(B, S, D, dtype):
    case(inputs(S, B, S, D, dtype, gates="i"), "variance")


@pytest.mark.parametrize("B,S,D", [(700, 3, 64), (300, 20, 70), (33, 40, 513), (1000, 1, 8)])
def test_many_sequences(B, S, D):
    case(inputs(S, B, S, D, "bf16"), "convex")


@pytest.mark.parametrize("B,S,D", [(513, 9, 65), (1100, 60, 33), (270000, 1, 2)])
def test_sums_of_the_rate_s_gradient_over_many_rows(B, S, D):
    """One, two and three passes over partial sums."""
    case(inputs(S, B, S, D, "f32", gates="", init=False), "convex", last=False)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rate,scale", [(False, "convex"), (False, None), (True, "variance"), (True, "convex")])
@pytest.mark.parametrize("gates", ["", "z", "iz"])
@pytest.mark.parametrize("D", [96, 95])
def test_many_units_with_every_gate(D, gates, rate, scale, dtype):
    case(inputs(D, 2, 1123, D, dtype, gates, rate), scale)


def test_strides_below_zero_in_the_c_interface():
    """Tokens from the last to the first, by a stride that runs backwards."""
    B, S, D = 2, 130, 64
    t = inputs(3, B, S, D, "bf16", gates="", rate=False, init=False, grad=False)
    dy = make(np.random.default_rng(4), B, S, D, dtype=BF16)
    back = {n: v.flip(1).contiguous() for n, v in (("x", t["x"]), ("f", t["f"]), ("dy", dy))}
    lib, st = _lib.load(), torch.cuda.current_stream().cuda_stream
    end = lambda v: v.data_ptr() + (S - 1) * D * 2  # noqa: E731
    strides = (ctypes.c_longlong * 8)(*[S * D, -D] * 2)
    y, ck, *grads = (torch.empty_like(t["x"]), torch.empty(lib.mlstm_b200_gated_checkpoint_bytes(B, S, D), dtype=torch.uint8, device="cuda"),
                     torch.empty_like(dy), torch.empty_like(dy))
    ws = torch.empty(lib.mlstm_b200_gated_workspace_bytes(B, S, D, 1), dtype=torch.uint8, device="cuda")
    fw = lib.mlstm_b200_gated_scan_fw(end(back["x"]), end(back["f"]), None, None, None, None, strides, y.data_ptr(), None, ck.data_ptr(), ws.data_ptr(),
                                      ws.numel(), B, S, D, 1, _lib.dtype_code(BF16), st)
    bw = lib.mlstm_b200_gated_scan_bw(end(back["x"]), end(back["f"]), None, None, None, strides, ck.data_ptr(), end(back["dy"]),
                                      (ctypes.c_longlong * 2)(S * D, -D), None, grads[0].data_ptr(), grads[1].data_ptr(), None, None, None, None,
                                      ws.data_ptr(), ws.numel(), B, S, D, 1, _lib.dtype_code(BF16), st)
    assert fw == bw == 0
    ref = O.gated_scan(x=f64(t["x"]), f=f64(t["f"]), input_scale="convex", dy=f64(dy))
    for got, n in zip((y, *grads), ("y", "dx", "df")):
        check(got, ref[n], n)


def test_strides():
    """Operands as parts of wider rows and with the batch inside, at offsets that no wide access fits too; the last axis apart; a gradient
    without memory of its own."""
    rng = np.random.default_rng(3)
    B, S, D = 3, 50, 40
    t = inputs(9, B, S, D, "bf16")
    for off in (0, 8, 2, 5):
        wide = make(rng, S, B, 200, dtype=BF16, grad=True).transpose(0, 1)
        rows = make(rng, B, S, 101, dtype=BF16, grad=True)
        t.update(x=wide[..., off:off + D], z=wide[..., 100 + off:100 + off + D], f=rows[..., off:off + D], i=rows[..., 50:50 + D])
        case(t, "variance")
    case(t, "variance", dy=torch.ones((), dtype=BF16, device="cuda").expand(B, S, D))
    t["f"] = make(rng, B, D, S, dtype=BF16, grad=True).transpose(1, 2)
    case(t, "convex", dy=make(rng, B, D, S, dtype=BF16).transpose(1, 2))


def test_operands_without_memory_of_their_own():
    """Gates the same for all sequences, for all tokens, for all channels: strides of zero, and gradients summed by whoever expanded them."""
    rng = np.random.default_rng(6)
    B, S, D = 3, 40, 24
    t = inputs(15, B, S, D, "f32", grad=False)
    t["f"], t["i"] = make(rng, 1, S, D).expand(B, S, D), make(rng, B, S, 1).expand(B, S, D)
    t["x"] = make(rng, B, 1, D).expand(B, S, D)
    case({n: v.requires_grad_(True) for n, v in t.items()}, "variance")


def test_one_tensor_in_several_places():
    """The same gate for what is kept and what is added: its gradient is the sum of both."""
    t = inputs(16, 2, 90, 48, "f32", gates="")
    both = dict(t, i=t["f"])
    dy = make(np.random.default_rng(1), 2, 90, 48)
    ref = O.gated_scan(**{n: f64(v) for n, v in both.items()}, dy=f64(dy))
    y = mk.gated_scan__b200(**both)
    g, = torch.autograd.grad(y, t["f"], dy)
    check(g, (ref["df"][0] + ref["di"][0], ref["df"][1] + ref["di"][1] + np.abs(ref["df"][0]) + np.abs(ref["di"][0])), "df + di")


def test_token_axis_of_any_stride():
    """One token, whose stride means nothing; and tokens further apart than 32 bits count."""
    rng = np.random.default_rng(4)
    t = inputs(3, 2, 1, 24, "f32")
    t["x"] = make(rng, 2, 24).as_strided((2, 1, 24), (24, 1 << 40, 1)).requires_grad_(True)
    case(t, "convex")
    t = inputs(3, 1, 2, 8, "bf16")
    far = torch.zeros((1 << 31) + 8, dtype=BF16, device="cuda")
    far[:8], far[-8:] = t["x"].detach()[0, 0], t["x"].detach()[0, 1]
    t["x"] = far.as_strided((1, 2, 8), (1 << 31, 1 << 31, 1)).requires_grad_(True)
    case(t, "convex")


def test_only_the_last_state_and_only_some_gradients():
    t = inputs(14, 2, 145, 40, "bf16")
    dh = make(np.random.default_rng(2), 2, 40)
    ref = O.gated_scan(**{n: f64(v) for n, v in t.items()}, input_scale="convex", dy=np.zeros((2, 145, 40)), dh_last=f64(dh))
    _, h = mk.gated_scan__b200(**t, input_scale="convex", return_last_states=True)
    for n, g in zip(t, torch.autograd.grad(h, list(t.values()), dh)):
        check(g, ref["d" + n], "d" + n)
    for n in ("f", "rate", "h_initial"):   # one input alone wants a gradient
        only = {m: v.detach().requires_grad_(m == n) for m, v in t.items()}
        _, h = mk.gated_scan__b200(**only, input_scale="convex", return_last_states=True)
        check(torch.autograd.grad(h, only[n], dh)[0], ref["d" + n], "d" + n)


def test_rate_and_state_in_16_bits():
    t = inputs(5, 2, 20, 32, "bf16")
    for n in ("rate", "h_initial"):
        t[n] = t[n].detach().bfloat16().requires_grad_(True)
    case(t, "variance")


# ---- where gates close and open -------------------------------------------------------------------------------------
@pytest.mark.parametrize("rate", [False, True])
@pytest.mark.parametrize("scale", SCALES)
@pytest.mark.parametrize("D", [64, 63])
def test_gates_far_open_and_far_closed(rate, scale, D):
    """Gates down to -60 and up to 60 of f32 inputs keep their digits, forward and backward."""
    rng = np.random.default_rng(D)
    t = inputs(17, 2, 150, D, "f32", rate=rate)
    with torch.no_grad():
        for n in ("f", "i", "z"):
            t[n].copy_(torch.from_numpy(rng.uniform(-60, 60, t[n].shape)))
    case(t, scale)


@pytest.mark.parametrize("scale", SCALES)
def test_long_memory(scale):
    """Rates of 1e-6 to 1: what a state forgets in a token has all its digits, however near one its factor is."""
    t = inputs(18, 1, 3000, 64, "f32", gates="", shift=0.0, init=False)
    with torch.no_grad():
        t["rate"].copy_(-torch.logspace(-6, 0, 64))
    case(t, scale)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("scale", SCALES)
def test_a_gate_of_minus_infinity_starts_anew(scale, dtype):
    t = inputs(19, 2, 300, 40, dtype, rate=False, grad=False)
    f = t["f"].clone()
    f[:, 130] = -float("inf")
    t = {n: v.requires_grad_(True) for n, v in {**t, "f": f}.items()}
    y, h = mk.gated_scan__b200(**t, input_scale=scale, return_last_states=True)
    cut = {n: v[:, 130:] for n, v in t.items() if n != "h_initial"}
    ref = O.gated_scan(**{n: f64(v) for n, v in cut.items()}, input_scale=scale)
    check(y[:, 130:], ref["y"], "y")
    check(h, ref["h_last"], "h")
    dy = torch.zeros_like(y)
    dy[:, 130:] = 1   # nothing goes back through a factor of zero
    for n, g in zip(t, torch.autograd.grad(y, list(t.values()), dy)):
        assert torch.isfinite(g).all(), n
        assert (g == 0).all() if n == "h_initial" else (g[:, :130] == 0).all(), n
    # whatever stood before it: an infinite state is left, too, only where its factor is not zero
    f2 = t["f"].detach().clone()
    f2[:, 130] = float("inf")
    y2 = mk.gated_scan__b200(**{**{n: v.detach() for n, v in t.items()}, "f": f2}, input_scale=scale)
    assert torch.isfinite(y2).all()


@pytest.mark.parametrize("scale", SCALES)
def test_closed_gates_give_numbers(scale):
    """1 - a and the input's scale vanish: f = 200 without a rate, f = -200 with one.  The state stays; gradients are numbers."""
    for f, rate in ((200.0, None), (-200.0, -0.5)):
        t = inputs(20, 2, 40, 16, "f32", rate=rate is not None)
        with torch.no_grad():
            t["f"].fill_(f)
        y, h = mk.gated_scan__b200(**t, input_scale=scale, return_last_states=True)
        if scale is not None:
            assert torch.equal(h, t["h_initial"])
        for n, g in zip(t, torch.autograd.grad((y, h), list(t.values()), (torch.ones_like(y), torch.ones_like(h)))):
            assert torch.isfinite(g).all(), n
            if n == "f" and scale is None:
                assert (g.abs() < 1e-30).all()


@pytest.mark.parametrize("B,S,D", [(2, 40, 32), (1, 700, 33)])
def test_nan_stays_in_its_channel(B, S, D):
    for n in TOKENS:
        t = inputs(2, B, S, D, "bf16", grad=False)
        t[n][-1, 5, 3] = float("nan")
        y, h = mk.gated_scan__b200(**t, input_scale="variance", return_last_states=True)
        bad = torch.zeros_like(y, dtype=torch.bool)
        if n == "z":
            bad[-1, 5, 3] = True
        else:
            bad[-1, 5:, 3] = True
        assert torch.equal(y.isnan(), bad)
        assert h.isnan().sum() == (0 if n == "z" else 1)


def test_rows_of_a_padded_batch():
    """What stands behind a sequence's end, NaN included, does not reach its outputs, nor the other sequences."""
    t = inputs(21, 3, 200, 64, "bf16", grad=False)
    y = mk.gated_scan__b200(**t, input_scale="convex")
    for n in TOKENS:
        t[n][1, 77:] = float("nan")
    y2 = mk.gated_scan__b200(**t, input_scale="convex")
    assert torch.equal(y[[0, 2]], y2[[0, 2]]) and torch.equal(y[1, :77], y2[1, :77])


# ---- tokens one by one ----------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("B,D", [(1, 8), (3, 65), (2, 96), (5, 1001), (2, 1000), (1, 1)])
@pytest.mark.parametrize("rate,scale", [(True, "variance"), (False, "convex"), (False, None)])
def test_tokens_one_by_one(B, D, dtype, rate, scale):
    """A prompt, then single tokens from its last state."""
    S = 12
    t = inputs(D, B, S, D, dtype, rate=rate, grad=False)
    ref = O.gated_scan(**{n: f64(v) for n, v in t.items()}, input_scale=scale)
    par = {"rate": t["rate"]} if rate else {}
    _, h = mk.gated_scan__b200(**{n: v[:, :5] if n in TOKENS else v for n, v in t.items()}, input_scale=scale, return_last_states=True)
    for s in range(5, S):
        now = {n: t[n][:, s] for n in TOKENS}
        old = h.clone()
        y, new = mk.gated_step__b200(**now, **par, h=h, input_scale=scale)
        assert torch.equal(h, old) and new.dtype == torch.float32
        check(y, (ref["y"][0][:, s], ref["y"][1][:, s]), "y")
        y2, same = mk.gated_step__b200(**now, **par, h=h, input_scale=scale, h_new=h)
        assert same is h and torch.equal(y, y2) and torch.equal(h, new)
    check(h, ref["h_last"], "h")


@pytest.mark.parametrize("gates", ["", "i", "z", "iz"])
def test_step_options(gates):
    for rate in (False, True):
        for scale in SCALES:
            for dtype in DTYPES:
                t = inputs(3, 70, 1, 264, dtype, gates, rate, grad=False)
                ref = O.gated_scan(**{n: f64(v) for n, v in t.items()}, input_scale=scale)
                y, h = mk.gated_step__b200(**{n: v[:, 0] if n in TOKENS else v for n, v in t.items() if n != "h_initial"}, h=t["h_initial"], input_scale=scale)
                check(y, (ref["y"][0][:, 0], ref["y"][1][:, 0]), "y")
                check(h, ref["h_last"], "h")


def test_step_of_strided_inputs_and_16_bit_states():
    """Parts of wider rows, an odd offset, a state in bf16: as the same call on copies."""
    rng = np.random.default_rng(2)
    rows = make(rng, 6, 400, dtype=BF16)
    for off in (0, 1):
        x, f, i, z = (rows[:, off + k * 96:off + k * 96 + 90] for k in range(4))
        h = make(rng, 6, 90, dtype=BF16)
        for a, b in zip(mk.gated_step__b200(x, f, h, i, z), mk.gated_step__b200(x.clone(), f.clone(), h.float(), i.clone(), z.clone())):
            assert torch.equal(a, b)


def test_buffers_that_overlap_are_refused():
    rng = np.random.default_rng(2)
    x, f, h = make(rng, 4, 32), make(rng, 4, 32), make(rng, 4, 32)
    with pytest.raises(ValueError, match="overlaps"):
        mk.gated_step__b200(x, f, h, h_new=x)
    big = make(rng, 5, 32)
    with pytest.raises(ValueError, match="overlaps"):
        mk.gated_step__b200(x, f, big[:4], h_new=big[1:])


# ---- streams, graphs, traces ----------------------------------------------------------------------------------------
def some_calls(grad=True):
    wide, deep = inputs(4, 2, 300, 64, "bf16", grad=grad), inputs(5, 1, 4100, 64, "f32", grad=grad)
    return {"wide": (lambda: mk.gated_scan__b200(**wide, input_scale="variance"), list(wide.values()), torch.ones(2, 300, 64, dtype=BF16, device="cuda")),
            "deep": (lambda: mk.gated_scan__b200(**deep, input_scale="convex"), list(deep.values()), torch.ones(1, 4100, 64, device="cuda"))}


@pytest.mark.parametrize("op", ["wide", "deep"])
def test_same_bits_again_on_another_stream_and_from_a_graph(op):
    fn, leaves, dy = some_calls()[op]

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
    jobs = some_calls().values()

    def run():
        out = []
        for fn, leaves, dy in jobs:
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


@pytest.mark.parametrize("op", ["wide", "deep"])
def test_compiled_without_graph_break(op):
    fn, leaves, dy = some_calls()[op]
    y = fn()
    eager = [y, *torch.autograd.grad(y, leaves, dy)]
    y = torch.compile(fn, fullgraph=True)()
    for a, b in zip(eager, [y, *torch.autograd.grad(y, leaves, dy)]):
        assert torch.equal(a, b)


def test_compiled_for_any_length():
    t = inputs(4, 2, 50, 64, "bf16", grad=False)
    fn = lambda t: mk.gated_scan__b200(**t, input_scale="variance", return_last_states=True)  # noqa: E731
    compiled = torch.compile(fn, fullgraph=True, dynamic=True)
    for S in (50, 33, 41):
        cut = {n: v[:, :S].contiguous() if n in TOKENS else v for n, v in t.items()}
        for a, b in zip(fn(cut), compiled(cut)):
            assert torch.equal(a, b)


def test_traced_operators_say_what_they_return():
    t = inputs(4, 2, 50, 64, "bf16", grad=False)
    args = [t[n] for n in ("x", "f", "i", "z", "rate", "h_initial")]
    test = ("test_schema", "test_faketensor")
    ops = torch.ops.mlstm_b200
    for keep in (False, True):
        for last in (False, True):
            torch.library.opcheck(ops.gated_scan, (*args, 2, keep, last), test_utils=test)
    _, _, ck = ops.gated_scan(*args, 2, True, True)
    torch.library.opcheck(ops.gated_scan_bw, (*args, 2, ck, t["x"], t["h_initial"]), test_utils=test)
    one = [v[:, 0] if v.dim() == 3 else v for v in args]
    torch.library.opcheck(ops.gated_step, (*one, 2), test_utils=test)
    torch.library.opcheck(ops.gated_step_into, (*one, 2, torch.empty_like(t["h_initial"])), test_utils=test)
    y, _, _ = ops.gated_scan(*(v.requires_grad_(True) for v in args), 0, False, False)
    with pytest.raises(RuntimeError, match="checkpoints"):
        y.sum().backward()


def test_steps_compile():
    t = inputs(4, 3, 1, 40, "bf16", grad=False)
    now = {n: t[n][:, 0] for n in TOKENS}

    def steps(h, h2):
        out = []
        for _ in range(2):
            y, g = mk.gated_step__b200(**now, rate=t["rate"], h=h, h_new=h2, input_scale="variance")
            y2, g2 = mk.gated_step__b200(**now, rate=t["rate"], h=g, input_scale="variance")
            assert g is h2
            out += [y, y2, g2]
            h, h2 = h2, h
        return out
    results = []
    for f in (steps, torch.compile(steps, fullgraph=True)):
        h, h2 = t["h_initial"].clone(), torch.empty_like(t["h_initial"])
        results.append([*f(h, h2), h, h2])
    for a, b in zip(*results):
        assert torch.equal(a, b)


def test_no_second_derivative():
    fn, leaves, _ = some_calls()["wide"]
    with pytest.raises(NotImplementedError, match="no second derivative"):
        torch.autograd.grad(fn().float().sum(), leaves, create_graph=True)


def test_no_tokens():
    z = lambda *s, **k: torch.zeros(*s, device="cuda", requires_grad=True)  # noqa: E731
    for B, S, D in ((2, 0, 8), (0, 3, 8), (0, 0, 8), (2, 3, 0)):
        x, rate, h0 = z(B, S, D), z(D), torch.ones(B, D, device="cuda", requires_grad=True)
        y, h = mk.gated_scan__b200(x, x, x, x, rate, h0, True)
        assert y.shape == x.shape and torch.equal(h, h0) and (h.numel() == 0 or h.data_ptr() != h0.data_ptr())
        gx, gr, g0 = torch.autograd.grad(h.sum() + y.sum(), (x, rate, h0))
        assert gx.shape == x.shape and (gr == 0).all() and (g0 == 1).all()
        assert (mk.gated_scan__b200(x, x, return_last_states=True)[1] == 0).all()
    y, h = mk.gated_step__b200(z(0, 8), z(0, 8), z(0, 8))
    assert y.shape == (0, 8) and h.shape == (0, 8)


def test_gradient_is_that_of_the_formula_by_differences():
    """Along a random direction of all inputs: the oracle's value there and back against the kernels' gradients."""
    for scale in SCALES:
        t = inputs(8, 2, 300, 12, "f32")
        rng = np.random.default_rng(2)
        w = make(rng, 2, 300, 12)
        grads = torch.autograd.grad(mk.gated_scan__b200(**t, input_scale=scale), list(t.values()), w)
        dirs = {n: rng.standard_normal(v.shape) for n, v in t.items()}
        loss = lambda s: (O.gated_scan(**{n: f64(v) + s * dirs[n] for n, v in t.items()}, input_scale=scale)["y"][0] * f64(w)).sum()  # noqa: E731
        d = (loss(1e-6) - loss(-1e-6)) / 2e-6
        terms = [(f64(g) * dirs[n]) for n, g in zip(t, grads)]
        size = sum(np.abs(v).sum() for v in terms)
        # of f32 gradients, each off by up to a few thousand units (decays over a few dozen tokens): 2^-12 of the absolute sum
        assert abs(d - sum(v.sum() for v in terms)) < size * 2.0 ** -12


def test_offsets_past_32_bits():
    """Tensors of more than 2^31 elements: the last sequence comes out as it does alone."""
    B, S, D = 521, 2048, 2048
    rng = np.random.default_rng(3)
    x = torch.zeros(B, S, D, dtype=BF16, device="cuda")
    assert x.numel() > 1 << 31
    x[-1] = make(rng, S, D, dtype=BF16)
    rate = -torch.exp(make(rng, D, shift=-2.0))

    def run(x):
        x = x.requires_grad_(True)
        y = mk.gated_scan__b200(x, x.detach(), rate=rate, input_scale="variance")
        g, = torch.autograd.grad(y, x, x.detach())
        return y[-1].detach().clone(), g[-1].clone()
    for got, alone in zip(run(x), run(x.detach()[-1:].clone())):
        # the sequence may be cut otherwise, which moves f32 values by some units and so a few bf16 ones by a step
        assert (got.float() - alone.float()).abs().max() <= 2.0 ** -7 * alone.float().abs().max()


def test_a_million_tokens():
    """In one call and in pieces that hand the state on: f32 roundings of some units a token (2^-22), over the few tokens that gates around a half
    remember (a below 0.99 in all but a few: 2^5 of them in sum), 2^-17 of the largest value.  And nothing waited in vain."""
    S, D = 1_000_003, 72
    gen = torch.Generator("cuda").manual_seed(3)
    x, f = (torch.randn(1, S, D, device="cuda", generator=gen) for _ in range(2))
    y, last = mk.gated_scan__b200(x, f, input_scale="convex", return_last_states=True)
    h, parts = None, []
    for at in range(0, S, 123457):
        p, h = mk.gated_scan__b200(x[:, at:at + 123457], f[:, at:at + 123457], h_initial=h, input_scale="convex", return_last_states=True)
        parts.append(p)
    assert (torch.cat(parts, 1) - y).abs().max() <= 2.0 ** -17 * y.abs().max()
    assert (h - last).abs().max() <= 2.0 ** -17 * y.abs().max()
    # The last state is that of joined runs (A h + H, a run's H added up from zero), the last output goes token by token from the state in
    # front of its run: two orders of the same at most eight roundings of 2^-24 and products of factors below 1, within the bound above.
    assert (last - y[:, -1]).abs().max() <= 2.0 ** -17 * y.abs().max()
    assert _lib.device_status() == 0


def test_launches_are_counted():
    t = inputs(4, 2, 300, 64, "bf16")
    n = _lib.launch_count()
    y = mk.gated_scan__b200(**t)
    assert _lib.launch_count() > n
    n = _lib.launch_count()
    torch.autograd.grad(y.sum(), t["x"])
    assert _lib.launch_count() > n
