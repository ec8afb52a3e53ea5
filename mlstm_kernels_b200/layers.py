"""The operators around a recurrence, in the layers that hold one: layer norm in front of it and of its heads' output, the short
causal convolution of its inputs, and the selective state space scan, a recurrence with a diagonal state beside the mLSTM's.

All run on CUDA tensors in f32, bf16 or f16 with sums and states in f32; tensors are read where they are as long as their last axis
is contiguous.  layer_norm__b200, short_conv__b200 and ssm_scan__b200 are differentiable (once); the *_step__b200 functions, for one
token at a time, are not.  They take the inputs' element types as they are, also inside an autocast region.  As with the other
functions of this package an eager call goes straight to the native host module (csrc/host_layers.cpp), and a traced one (torch.compile)
through the custom operators of _ops.py.  A backward pass can be captured in a CUDA graph as long as no
autograd graph of the same leaves is alive outside the capture (PyTorch's rule for every operator: it would wait for that graph's
stream, which ends the capture).
"""

from __future__ import annotations

import torch

from . import _lib, _ops


def _silu(activation: str | None) -> bool:
    if activation not in (None, "silu"):
        raise ValueError(f"Unsupported activation {activation!r}: None or 'silu'.")
    return activation == "silu"


def layer_norm__b200(
    x: torch.Tensor,  # (..., D), or (..., NH, D) with weight (NH, D)
    weight: torch.Tensor = None,  # (D,) or (NH, D)
    bias: torch.Tensor = None,  # as weight
    eps: float = 1e-6,
) -> torch.Tensor:
    """(x - mean) / sqrt(var + eps) * weight + bias over the last axis (at most 16384 elements), in x's dtype.

    weight and bias may be f32 next to x in 16 bits.  With weights (NH, D) every head has its own: the output of a recurrence,
    (B, NH, S, D), is passed as h.transpose(1, 2) and read in place, and its gradient comes back in h's own layout."""
    if torch.compiler.is_compiling():
        return _ops.layer_norm(x, weight, bias, eps)[0]
    return _lib.host().layer_norm(x, weight, bias, eps)


def short_conv__b200(
    x: torch.Tensor,  # (B, S, D)
    weight: torch.Tensor,  # (D, W), W = 2, 3 or 4; the last tap is the token's own
    bias: torch.Tensor = None,  # (D,)
    x_initial: torch.Tensor = None,  # (B, W - 1, D): the tokens before the first (zeros without)
    return_last_states: bool = False,
    activation: str = None,  # None or "silu"
):
    """act(bias + sum_j weight[:, j] x[t - W + 1 + j]) for every channel; with return_last_states also the last W - 1 tokens
    (B, W - 1, D), which the next call takes as x_initial and short_conv_step__b200 as its state."""
    silu = _silu(activation)
    if torch.compiler.is_compiling():
        y, last = _ops.short_conv(x, weight, bias, x_initial, return_last_states, silu)
    else:
        y, last = _lib.host().short_conv(x, weight, bias, x_initial, return_last_states, silu)
    return (y, last) if return_last_states else y


def short_conv_step__b200(
    x: torch.Tensor,  # (B, D)
    state: torch.Tensor,  # (B, W - 1, D): the tokens before
    weight: torch.Tensor,  # (D, W)
    bias: torch.Tensor = None,  # (D,)
    activation: str = None,
    state_new: torch.Tensor = None,  # optional buffer for the new state: `state` itself, or apart from all that is read
) -> tuple[torch.Tensor, torch.Tensor]:
    """One token of short_conv__b200: returns y (B, D) and the new state; the old state is untouched unless it is state_new."""
    silu = _silu(activation)
    if torch.compiler.is_compiling():
        if state_new is None:
            return _ops.short_conv_step(x, state, weight, bias, silu)
        return _ops.short_conv_step_into(x, state, weight, bias, silu, state_new), state_new
    return _lib.host().short_conv_step(x, state, weight, bias, silu, state_new)


def ssm_scan__b200(
    x: torch.Tensor,  # (B, S, D)
    dt: torch.Tensor,  # (B, S, D)
    a: torch.Tensor,  # (D, N), N <= 128
    b: torch.Tensor,  # (B, S, N) or (B, S, G, N)
    c: torch.Tensor,  # as b
    skip: torch.Tensor = None,  # (D,)
    z: torch.Tensor = None,  # (B, S, D)
    dt_bias: torch.Tensor = None,  # (D,)
    softplus: bool = False,
    h_initial: torch.Tensor = None,  # (B, D, N) (zeros without)
    return_last_states: bool = False,
):
    """Selective state space scan, N states to a channel:

        step_t = softplus(dt_t + dt_bias) (or dt_t + dt_bias);   h_t = exp(step_t a) h_{t-1} + step_t x_t b_t
        y_t = (c_t . h_t + skip x_t) silu(z_t)

    x, dt, b, c, z share one dtype, that of y.  With G groups, group g of b and c belongs to the channels g D/G ... (g+1) D/G - 1.
    With return_last_states also the state after the last token, (B, D, N) in f32, which the next call takes as h_initial and
    ssm_step__b200 as its state.  Rows of a padded batch do not touch each other, and outputs in front of the padding do not see it;
    the last state does.  An infinity in x or dt may leave infinities or NaN in its channel from there on."""
    if torch.compiler.is_compiling():
        keep = torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, dt, a, b, c, skip, z, dt_bias, h_initial))
        y, last, _ = _ops.ssm_scan(x, dt, a, b, c, skip, z, dt_bias, softplus, h_initial, keep, bool(return_last_states))
    else:
        y, last = _lib.host().ssm_scan(x, dt, a, b, c, skip, z, dt_bias, h_initial, softplus, return_last_states)
    return (y, last) if return_last_states else y


def ssm_step__b200(
    x: torch.Tensor,  # (B, D)
    dt: torch.Tensor,  # (B, D)
    a: torch.Tensor,  # (D, N)
    b: torch.Tensor,  # (B, N) or (B, G, N)
    c: torch.Tensor,
    h: torch.Tensor,  # (B, D, N)
    skip: torch.Tensor = None,
    z: torch.Tensor = None,  # (B, D)
    dt_bias: torch.Tensor = None,
    softplus: bool = False,
    h_new: torch.Tensor = None,  # optional f32 buffer for the new state: `h` itself, or apart from all that is read
) -> tuple[torch.Tensor, torch.Tensor]:
    """One token of ssm_scan__b200: returns y (B, D) and the new state in f32; the old state is untouched unless it is h_new."""
    if torch.compiler.is_compiling():
        if h_new is None:
            return _ops.ssm_step(x, dt, a, b, c, h, skip, z, dt_bias, softplus)
        return _ops.ssm_step_into(x, dt, a, b, c, h, skip, z, dt_bias, softplus, h_new), h_new
    return _lib.host().ssm_step(x, dt, a, b, c, skip, z, dt_bias, h, softplus, h_new)
