"""Helpers for the tests of the operators around a recurrence: inputs rounded to their element type, and results compared with the
oracle's values within its bound on f32 arithmetic and half a step of the result's type."""

import numpy as np
import torch

TDT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SMALLEST = {torch.float32: 2.0 ** -126, torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -24}   # steps near zero


def make(rng, *shape, dtype=torch.float32, scale=1.0, shift=0.0, grad=False):
    t = torch.from_numpy(np.asarray(rng.standard_normal(shape) * scale + shift)).to(dtype).cuda()
    return t.requires_grad_(True) if grad else t


def f64(t):
    return None if t is None else t.detach().double().cpu().numpy()


def check(got, ref, name=""):
    """got: tensor; ref: (value, bound in units of 2^-24) of the oracle."""
    value, units = ref
    assert tuple(got.shape) == value.shape, (name, got.shape, value.shape)
    g = f64(got)
    assert np.isfinite(g).all(), name
    half = torch.finfo(got.dtype).eps / 2
    f32 = units * 2.0 ** -24
    tol = f32 + half * (np.abs(value) + f32) + SMALLEST[got.dtype]
    worst = (np.abs(g - value) / np.maximum(tol, 1e-300)).max() if value.size else 0.0
    assert worst <= 1, (name, worst)
