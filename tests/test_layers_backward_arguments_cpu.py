"""The backward operators of traced models take what their forward operators gave and nothing else: gradients, statistics and
checkpoints of another size or type are refused before anything is launched.  On fake CUDA tensors, without a GPU."""

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

from mlstm_kernels_b200 import _lib

B, S, D, N, NH = 2, 40, 24, 16, 3
F32, BF16 = torch.float32, torch.bfloat16


def e(*shape, dt=BF16):
    return torch.empty(*shape, dtype=dt, device="cuda")


def refused(fn, args, name, value, kind=ValueError):
    with pytest.raises(kind, match="layer_norm__b200|short_conv__b200|ssm_scan__b200|CUDA tensors only"):
        fn(*{**args, name: value}.values())


@pytest.mark.parametrize("heads", [False, True])
def test_norm(heads):
    fn = _lib.host().layer_norm_bw
    with FakeTensorMode():
        a = dict(x=e(B, S, NH, D), weight=e(NH, D, dt=F32) if heads else e(D, dt=F32), mean=e(B * S * NH, dt=F32), rstd=e(B * S * NH, dt=F32),
                 dy=e(B, S, NH, D), heads=heads, param_dtype=F32, want_w=True, want_b=True)
        for name, value in (("mean", e(B * S, dt=F32)), ("rstd", e(B * S * NH - 1, dt=F32)), ("mean", e(B * S * NH, dt=BF16)), ("rstd", e(2 * B * S * NH, dt=F32)[::2]),
                            ("dy", e(B, S, NH, D - 1)), ("dy", e(B * S, NH, D)), ("heads", not heads), ("param_dtype", BF16), ("param_dtype", torch.float64)):
            refused(fn, a, name, value)
        refused(fn, {**a, "weight": None}, "param_dtype", torch.int32)
        refused(fn, a, "dy", torch.empty(B, S, NH, D, dtype=BF16), RuntimeError)


def test_conv():
    fn = _lib.host().short_conv_bw
    with FakeTensorMode():
        a = dict(x=e(B, S, D), weight=e(D, 4), bias=e(D), x_initial=e(B, 3, D), dy=e(B, S, D), dx_last=e(B, 3, D), silu=True, want_w=True, want_b=True,
                 want_initial=True)
        for name, value in (("dy", e(B, S - 1, D)), ("dy", e(B * S, D)), ("dx_last", e(B, 4, D)), ("dx_last", e(B, S, D))):
            refused(fn, a, name, value)


def test_scan():
    fn = _lib.host().ssm_scan_bw
    need = _lib.load().mlstm_b200_ssm_checkpoint_bytes(B, S, D, N)
    with FakeTensorMode():
        a = dict(x=e(B, S, D), dt=e(B, S, D), a=e(D, N, dt=F32), b=e(B, S, N), c=e(B, S, N), skip=None, z=None, dt_bias=None, h=None, softplus=True,
                 checkpoints=e(need, dt=torch.uint8), dy=e(B, S, D), dh_last=e(B, D, N, dt=F32))
        for name, value in (("checkpoints", e(need - 1, dt=torch.uint8)), ("checkpoints", e(0, dt=torch.uint8)), ("checkpoints", e(2 * need, dt=torch.uint8)[::2]),
                            ("dy", e(B, S, D + 1)), ("dy", e(B, D)), ("dh_last", e(B, D, N + 1, dt=F32)), ("dh_last", e(B, N, dt=F32))):
            refused(fn, a, name, value)
