"""Malformed calls of the gated linear recurrence and of dropout are refused before anything is launched: checked without a GPU, on fake
CUDA tensors, and through the C ABI with pointers that are never read."""

import ctypes

import pytest
import torch
import torch.autograd.forward_ad as fwAD
from torch._subclasses.fake_tensor import FakeTensorMode

import mlstm_kernels_b200 as mk
from mlstm_kernels_b200 import _lib

B, S, D = 2, 5, 24
F32, BF16 = torch.float32, torch.bfloat16


def e(*shape, dt=BF16, dev="cuda"):
    return torch.empty(*shape, dtype=dt, device=dev)


OPS = {
    "scan": (mk.gated_scan__b200, lambda: dict(x=e(B, S, D), f=e(B, S, D), i=e(B, S, D), z=e(B, S, D), rate=e(D, dt=F32), h_initial=e(B, D, dt=F32))),
    "step": (mk.gated_step__b200, lambda: dict(x=e(B, D), f=e(B, D), h=e(B, D, dt=F32), i=e(B, D), z=e(B, D), rate=e(D, dt=F32), h_new=e(B, D, dt=F32))),
    "dropout": (lambda x, residual, seed=3: mk.dropout__b200(x, 0.1, seed, residual=residual), lambda: dict(x=e(B, S, D), residual=e(B, S, D))),
}
EVERY = [(op, name) for op, (_, args) in OPS.items() for name in {"scan": ("x", "f", "i", "z", "rate", "h_initial"),
         "step": ("x", "f", "h", "i", "z", "rate", "h_new"), "dropout": ("x", "residual")}[op]]


@pytest.mark.parametrize("op,name", EVERY)
def test_wrong_shapes(op, name):
    fn, args = OPS[op]
    with FakeTensorMode():
        for change in (lambda s: (*s[:-1], s[-1] + 1), lambda s: (s[0] + 1, *s[1:]), lambda s: (1, 1, *s), lambda s: (1,)):
            a = args()
            a[name] = e(*change(tuple(a[name].shape)), dt=a[name].dtype)
            with pytest.raises(ValueError, match="shape|must be"):
                fn(**a)


@pytest.mark.parametrize("op,name", EVERY)
def test_host_memory_and_types(op, name):
    fn, args = OPS[op]
    with FakeTensorMode():
        a = args()
        a[name] = e(*a[name].shape, dt=a[name].dtype, dev="cpu")
        with pytest.raises(RuntimeError, match="CUDA tensors only"):
            fn(**a)
        a = args()
        a[name] = e(*a[name].shape, dt=torch.float64)
        with pytest.raises(ValueError, match="dtype|f32"):
            fn(**a)
        a = args()
        a[name] = e(*a[name].shape, dt=a[name].dtype, dev="cuda:1")
        with pytest.raises(ValueError, match="different devices"):
            fn(**a)
        if name in ("x", "f", "h"):
            with pytest.raises(TypeError, match="must be a tensor"):
                fn(**{**args(), name: None})
        with pytest.raises(TypeError, match="must be a tensor"):
            fn(**{**args(), name: 1.0})


@pytest.mark.parametrize("op,name", [(o, n) for o, n in EVERY if n not in ("h_new",)])
def test_forward_mode_tangents(op, name):
    fn, args = OPS[op]
    with FakeTensorMode(), fwAD.dual_level():
        a = args()
        a[name] = fwAD.make_dual(a[name], torch.empty_like(a[name]))
        with pytest.raises(NotImplementedError, match="forward-mode"):
            fn(**a)


def test_mixed_types():
    with FakeTensorMode():
        for op, name, dt in (("scan", "f", F32), ("scan", "i", torch.float16), ("scan", "z", F32), ("step", "f", F32), ("step", "h_new", BF16),
                             ("dropout", "residual", torch.float16)):
            fn, args = OPS[op]
            a = args()
            a[name] = e(*a[name].shape, dt=dt)
            with pytest.raises(ValueError, match="dtype|f32"):
                fn(**a)
        with pytest.raises(ValueError, match="dtype"):
            mk.dropout__b200(e(B, D, dt=F32), 0.1, 1, residual=e(B, D))   # a residual of fewer bits than x


def test_other_limits():
    with FakeTensorMode():
        for scale in ("Convex", "", 0, True):
            with pytest.raises(ValueError, match="Unsupported input_scale"):
                mk.gated_scan__b200(e(B, S, D), e(B, S, D), input_scale=scale)
        for scale in (-1, 3):
            with pytest.raises(ValueError, match="Unsupported input scale"):
                _lib.host().gated_scan(e(B, S, D), e(B, S, D), None, None, None, None, scale, False)
        with pytest.raises(ValueError, match="2\\^30"):
            mk.gated_scan__b200(e(1, (1 << 30) + 1, 8), e(1, (1 << 30) + 1, 8))
        with pytest.raises(ValueError, match="contiguous"):
            mk.gated_step__b200(e(B, D), e(B, D), e(B, D, dt=F32), h_new=e(D, B, dt=F32).t())
        for p in (-0.1, 1.5, float("nan"), float("inf")):
            with pytest.raises(ValueError, match="from 0 to 1"):
                mk.dropout__b200(e(B, D), p, 1)
        with pytest.raises(ValueError, match="negative"):
            mk.dropout__b200(e(B, D), 0.1, -1)
        with pytest.raises(ValueError, match="negative"):
            mk.dropout__b200(e(B, D), 0.1, 1, offset=-5)
        with pytest.raises(OverflowError):
            mk.dropout__b200(e(B, D), 0.1, 1 << 64)
        for seed in (1.5, None, "1"):
            with pytest.raises(TypeError):
                mk.dropout__b200(e(B, D), 0.1, seed)
        for seed in (e(1, dt=torch.int32), e(2, dt=torch.int64), e(0, dt=torch.int64), e(1, dt=F32)):
            with pytest.raises(ValueError, match="seed must be"):
                mk.dropout__b200(e(B, D), 0.1, seed)
        with pytest.raises(RuntimeError, match="CUDA tensors only"):
            mk.dropout__b200(e(B, D), 0.1, e(1, dt=torch.int64, dev="cpu"))
        with pytest.raises(ValueError, match="different devices"):
            mk.dropout__b200(e(B, D), 0.1, e(1, dt=torch.int64, dev="cuda:1"))


def test_backward_operators():
    """What is not what the forward gave is refused: gradients and checkpoints of another size or type."""
    scan_bw, drop_bw = _lib.host().gated_scan_bw, _lib.host().dropout_bw
    need = _lib.load().mlstm_b200_gated_checkpoint_bytes(B, S, D)
    with FakeTensorMode():
        a = dict(x=e(B, S, D), f=e(B, S, D), i=None, z=None, rate=None, h=None, scale=0, checkpoints=e(max(need, 256), dt=torch.uint8), dy=e(B, S, D),
                 dh_last=e(B, D, dt=F32))
        for name, value in (("checkpoints", e(need - 1, dt=torch.uint8)), ("checkpoints", e(0, dt=torch.uint8)), ("checkpoints", e(2 * need, dt=torch.uint8)[::2]),
                            ("dy", e(B, S, D + 1)), ("dy", e(B, D)), ("dh_last", e(B, D + 1, dt=F32)), ("dh_last", e(D, dt=F32))):
            with pytest.raises(ValueError, match="gated_scan__b200"):
                scan_bw(*{**a, name: value}.values())
        for dy, dt in ((e(B, D), torch.float64), (e(B, D), F32), (e(B, D), torch.float16)):
            with pytest.raises(ValueError, match="dropout__b200"):
                drop_bw(dy, None, 1, 0.1, 0, dt)


@pytest.mark.parametrize("B,S,D", [(2, 100, 24), (1, 16, 7), (3, 17, 65), (1, 1, 1)])
def test_what_the_traced_operators_say(B, S, D):
    with FakeTensorMode():
        x = e(B, S, D)
        y, h, ck = torch.ops.mlstm_b200.gated_scan(x, x, None, None, None, None, 1, True, True)
        assert y.shape == x.shape and y.dtype == BF16 and h.shape == (B, D) and h.dtype == F32
        assert ck.numel() == max(256, _lib.load().mlstm_b200_gated_checkpoint_bytes(B, S, D))
        assert torch.ops.mlstm_b200.dropout(x, None, None, 1, 0.1, 0).dtype == BF16
        assert torch.ops.mlstm_b200.dropout(x, e(B, S, D, dt=F32), None, 1, 0.1, 0).dtype == F32


def test_c_abi():
    lib = _lib.load()
    st = (ctypes.c_longlong * 8)(*([1] * 8))
    sizes = lambda *n: (ctypes.c_longlong * 4)(*n)  # noqa: E731
    p = ctypes.c_void_p(1 << 20)   # never read: every call below is refused first
    odd = ctypes.c_void_p((1 << 20) + 4)
    n = None
    assert lib.mlstm_b200_gated_checkpoint_bytes(0, 1, 8) == lib.mlstm_b200_gated_workspace_bytes(1, 0, 8, 1) == 0
    need = lib.mlstm_b200_gated_workspace_bytes(1, 500, 8, 0)
    fw = lambda S=500, scale=0, dt=1, f=p, ck=n, ws=p, size=need: lib.mlstm_b200_gated_scan_fw(p, f, n, n, n, n, st, p, n, ck, ws, size, 1, S, 8, scale, dt, n)  # noqa: E731
    assert need > 0 and lib.mlstm_b200_gated_workspace_bytes(1, 56, 8, 0) == 0   # one unit of work: nothing to hand on
    assert fw(0) == -1 and fw(scale=3) == -1 and fw(scale=-1) == -1 and fw(dt=7) == -2 and fw(f=n) == -3 and fw(ck=odd) == -4
    assert fw(ws=n) == -3 and fw(ws=odd) == -4 and fw(size=need - 1) == -5
    need = lib.mlstm_b200_gated_workspace_bytes(2, 100, 8, 1)

    def bw(i=n, z=n, rate=n, ck=p, di=n, dz=n, drate=n, ws=p, size=need, dt=1):
        return lib.mlstm_b200_gated_scan_bw(p, p, i, z, rate, st, ck, p, st, n, p, p, di, dz, drate, n, ws, size, 2, 100, 8, 1, dt, n)
    assert bw(i=p) == -3 and bw(z=p) == -3 and bw(di=p) == -3 and bw(dz=p) == -3 and bw(ck=n) == -3 and bw(dt=9) == -2 and bw(ck=odd) == -4
    assert need > 0 and bw(size=need - 1) == -5 and bw(ws=n) == -3 and bw(drate=p) == -3 and bw(ws=odd) == -4
    assert lib.mlstm_b200_gated_step(p, p, n, n, n, n, p, p, 1, 8, 0, 1, n) == -3 and lib.mlstm_b200_gated_step(p, p, n, n, n, p, p, p, 0, 8, 0, 1, n) == -1

    def drop(n4=(1, 1, 1, 8), prob=0.1, x=p, dt=1, odt=1, res=n, rst=n):
        return lib.mlstm_b200_dropout(x, st, res, rst, p, st, sizes(*n4), prob, 1, n, 0, dt, odt, n)
    assert drop(x=n) == -3 and drop(res=p) == -3 and drop(dt=1, odt=2) == -2 and drop(dt=5) == -2 and drop(prob=1.1) == -1 and drop(prob=float("nan")) == -1
    assert drop(n4=(0, 1, 1, 8)) == -1 and drop(n4=(1 << 20, 1 << 20, 1, 8)) == -1 and drop(n4=(1, -1, 1, 8)) == -1
