"""Malformed calls of the operators around a recurrence are refused before anything is launched: checked without a GPU, on fake CUDA
tensors, and through the C ABI with null pointers."""

import ctypes

import pytest
import torch
import torch.autograd.forward_ad as fwAD
from torch._subclasses.fake_tensor import FakeTensorMode

import mlstm_kernels_b200 as mk
from mlstm_kernels_b200 import _lib

B, S, D, N, G, W, NH = 2, 5, 24, 16, 3, 4, 4


def e(*shape, dt=torch.bfloat16, dev="cuda"):
    return torch.empty(*shape, dtype=dt, device=dev)


F32 = torch.float32
OPS = {
    "norm": (mk.layer_norm__b200, lambda: dict(x=e(B, S, NH, D), weight=e(NH, D, dt=F32), bias=e(NH, D, dt=F32))),
    "conv": (mk.short_conv__b200, lambda: dict(x=e(B, S, D), weight=e(D, W), bias=e(D), x_initial=e(B, W - 1, D))),
    "conv_step": (mk.short_conv_step__b200, lambda: dict(x=e(B, D), state=e(B, W - 1, D), weight=e(D, W), bias=e(D), state_new=e(B, W - 1, D))),
    "ssm": (mk.ssm_scan__b200, lambda: dict(x=e(B, S, D), dt=e(B, S, D), a=e(D, N, dt=F32), b=e(B, S, G, N), c=e(B, S, G, N), skip=e(D, dt=F32),
                                            z=e(B, S, D), dt_bias=e(D, dt=F32), h_initial=e(B, D, N, dt=F32))),
    "ssm_step": (mk.ssm_step__b200, lambda: dict(x=e(B, D), dt=e(B, D), a=e(D, N, dt=F32), b=e(B, G, N), c=e(B, G, N), h=e(B, D, N, dt=F32),
                                                 skip=e(D, dt=F32), z=e(B, D), dt_bias=e(D, dt=F32), h_new=e(B, D, N, dt=F32))),
}
EVERY = [(op, name) for op, (_, args) in OPS.items() for name in {"norm": ("x", "weight", "bias"), "conv": ("x", "weight", "bias", "x_initial"),
         "conv_step": ("x", "state", "weight", "bias", "state_new"), "ssm": ("x", "dt", "a", "b", "c", "skip", "z", "dt_bias", "h_initial"),
         "ssm_step": ("x", "dt", "a", "b", "c", "h", "skip", "z", "dt_bias", "h_new")}[op]]


@pytest.mark.parametrize("op,name", EVERY)
def test_wrong_shapes(op, name):
    fn, args = OPS[op]
    with FakeTensorMode():
        for change in (lambda s: (*s[:-1], s[-1] + 1), lambda s: (s[0] + 1, *s[1:]), lambda s: (1, 1, *s), lambda s: (1,)):
            a = args()
            shape = change(tuple(a[name].shape))
            if op == "norm" and name == "x" and len(shape) >= 2 and shape[-2:] == (NH, D):
                continue   # another number of rows is another call
            a[name] = e(*shape, dt=a[name].dtype)
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
    if name not in ("bias", "x_initial", "state_new", "skip", "z", "dt_bias", "h_initial", "h_new") and (op, name) != ("norm", "weight"):
        with FakeTensorMode(), pytest.raises(TypeError, match="must be a tensor"):
            fn(**{**args(), name: None})
    with FakeTensorMode(), pytest.raises(TypeError, match="must be a tensor"):
        fn(**{**args(), name: 1.0})


@pytest.mark.parametrize("op,name", [(o, n) for o, n in EVERY if o in ("norm", "conv", "ssm")])
def test_forward_mode_tangents(op, name):
    fn, args = OPS[op]
    with FakeTensorMode(), fwAD.dual_level():
        a = args()
        a[name] = fwAD.make_dual(a[name], torch.empty_like(a[name]))
        with pytest.raises(NotImplementedError, match="forward-mode"):
            fn(**a)


def test_mixed_types():
    with FakeTensorMode():
        for op, name, dt in (("norm", "bias", torch.bfloat16), ("conv", "bias", F32), ("conv", "x_initial", F32), ("conv_step", "state", torch.float16),
                             ("ssm", "dt", F32), ("ssm", "z", torch.float16), ("ssm_step", "b", F32), ("conv_step", "state_new", F32),
                             ("ssm_step", "h_new", torch.bfloat16)):
            fn, args = OPS[op]
            a = args()
            a[name] = e(*a[name].shape, dt=dt)
            with pytest.raises(ValueError, match="dtype|f32"):
                fn(**a)


def test_other_limits():
    with FakeTensorMode():
        for taps in (0, 1, 5):
            with pytest.raises(ValueError, match="2 to 4 taps"):
                mk.short_conv__b200(e(B, S, D), e(D, taps))
        with pytest.raises(ValueError, match="16384"):
            mk.layer_norm__b200(e(3, 16385))
        with pytest.raises(ValueError, match="N from 1 to 128"):
            mk.ssm_scan__b200(e(B, S, D), e(B, S, D), e(D, 129, dt=F32), e(B, S, 129), e(B, S, 129))
        with pytest.raises(ValueError, match="multiple of G"):
            mk.ssm_scan__b200(e(B, S, D), e(B, S, D), e(D, N, dt=F32), e(B, S, 5, N), e(B, S, 5, N))
        with pytest.raises(ValueError, match="2\\^30"):
            mk.short_conv__b200(e(1, (1 << 30) + 1, 8), e(8, 4))
        with pytest.raises(ValueError, match="Unsupported activation"):
            mk.short_conv__b200(e(B, S, D), e(D, 4), activation="gelu")
        a = OPS["conv_step"][1]()
        a["state_new"] = e(B, D, W - 1).transpose(1, 2)
        with pytest.raises(ValueError, match="contiguous"):
            mk.short_conv_step__b200(**a)


@pytest.mark.parametrize("B,S,D,N", [(2, 100, 24, 16), (1, 16, 7, 1), (3, 17, 65, 33), (1, 1, 1, 128)])
def test_checkpoints_of_the_traced_operator(B, S, D, N):
    """The traced operator's own count of the checkpoints' bytes is the library's."""
    with FakeTensorMode():
        x, bc = e(B, S, D), e(B, S, N)
        y, h, ck = torch.ops.mlstm_b200.ssm_scan(x, x, e(D, N, dt=F32), bc, bc, None, None, None, True, None)
    assert y.shape == (B, S, D) and h.shape == (B, D, N) and h.dtype == F32
    assert ck.numel() == max(256, _lib.load().mlstm_b200_ssm_checkpoint_bytes(B, S, D, N))


def test_c_abi():
    lib = _lib.load()
    st = (ctypes.c_longlong * 12)(*([1] * 12))
    p = ctypes.c_void_p(1 << 20)   # never read: every call below is refused first
    odd = ctypes.c_void_p((1 << 20) + 4)
    n = None
    assert lib.mlstm_b200_layer_norm_fw(p, st, n, n, p, n, n, 1, 1, 1, 16385, 1, 1, 1e-6, n) == -1
    assert lib.mlstm_b200_layer_norm_fw(p, st, n, n, p, n, n, 0, 1, 1, 64, 1, 1, 1e-6, n) == -1
    assert lib.mlstm_b200_layer_norm_fw(p, st, n, n, p, n, n, 1, 1, 1, 64, 7, 1, 1e-6, n) == -2
    assert lib.mlstm_b200_layer_norm_fw(p, st, n, n, n, n, n, 1, 1, 1, 64, 1, 1, 1e-6, n) == -3
    assert lib.mlstm_b200_layer_norm_fw(p, st, n, n, p, p, n, 1, 1, 1, 64, 1, 1, 1e-6, n) == -3
    need = lib.mlstm_b200_layer_norm_bw_workspace_bytes(100, 2, 64)
    bw = lambda ws, size: lib.mlstm_b200_layer_norm_bw(p, st, p, p, p, p, st, p, st, p, p, ws, size, 10, 10, 2, 64, 1, 0, n)  # noqa: E731
    assert need > 0 and bw(p, need - 1) == -5 and bw(odd, need) == -4 and bw(n, 0) == -3
    assert lib.mlstm_b200_short_conv_fw(p, st, n, p, n, p, n, 1, 1, 8, 5, 0, 1, 1, n) == -1
    assert lib.mlstm_b200_short_conv_fw(p, st, n, n, n, p, n, 1, 1, 8, 4, 0, 1, 1, n) == -3
    assert lib.mlstm_b200_short_conv_step(p, p, p, n, p, n, 1, 8, 4, 0, 1, 1, n) == -3
    need = lib.mlstm_b200_short_conv_bw_workspace_bytes(2, 100, 8, 4)
    bw = lambda ws, size: lib.mlstm_b200_short_conv_bw(p, st, n, p, n, p, st, n, p, n, p, n, ws, size, 2, 100, 8, 4, 1, 1, 1, n)  # noqa: E731
    assert need > 0 and bw(p, need - 1) == -5 and bw(odd, need) == -4 and bw(n, 0) == -3
    assert lib.mlstm_b200_ssm_checkpoint_bytes(1, 16, 8, 129) == 0 and lib.mlstm_b200_ssm_workspace_bytes(1, 16, 9, 16, 2, 1) == 0
    fw = lambda D, N, G, ws, size, ck=n: lib.mlstm_b200_ssm_scan_fw(p, p, p, p, p, n, n, n, n, st, p, n, ck, ws, size, 1, 4096, D, N, G, 1, 1, n)  # noqa: E731
    need = lib.mlstm_b200_ssm_workspace_bytes(1, 4096, 64, 16, 1, 0)
    assert need > 0 and fw(64, 16, 1, p, need - 1) == -5 and fw(64, 16, 1, n, 0) == -3 and fw(64, 16, 1, p, need, odd) == -4
    assert fw(64, 129, 1, p, need) == -1 and fw(64, 16, 5, p, need) == -1
    far = (ctypes.c_longlong * 12)(*([1] * 7 + [1 << 29] + [1] * 4))
    assert lib.mlstm_b200_ssm_scan_fw(p, p, p, p, p, n, n, n, n, far, p, n, n, p, need, 1, 4096, 64, 16, 1, 1, 1, n) == -1
    need = lib.mlstm_b200_ssm_workspace_bytes(1, 4096, 64, 16, 1, 1)
    bw = lambda dz, ws, size: lib.mlstm_b200_ssm_scan_bw(p, p, p, p, p, n, p, n, st, p, p, st, n, p, p, p, p, p, n, dz, n, n, ws, size, 1, 4096, 64, 16, 1, 1, 1,  # noqa: E731
                                                         n)
    assert bw(n, p, need) == -3 and bw(p, p, need - 1) == -5 and bw(p, odd, need) == -4
    assert lib.mlstm_b200_ssm_step(p, p, p, p, p, n, n, n, n, p, p, 1, 64, 16, 1, 1, 1, n) == -3
    assert lib.mlstm_b200_ssm_step(p, p, p, p, p, n, n, n, p, p, p, 1, 64, 16, 5, 1, 1, n) == -1
