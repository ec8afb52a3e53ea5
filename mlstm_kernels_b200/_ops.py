"""The kernels as PyTorch custom operators, for callers that trace their models (torch.compile).

The eager shims of chunkwise.py / recurrent.py talk to the shared library through ctypes, which a tracer can neither
follow nor skip.  Wrapped as `torch.library` operators the same calls become opaque nodes of the traced graph: shapes
and dtypes of the outputs come from the `register_fake` functions below (which only ask the library host-side
questions - chunk size, state element type, workspace size), gradients from `register_autograd`.  The reference's
Triton kernels are traceable in the same sense (its benchmark compiles whole models:
mlstm_kernels/utils/benchmark/benchmarks/interface.py:94-95).

The public functions switch to these operators only while a trace is being taken (`torch.compiler.is_compiling()`);
eager calls keep the direct path, which costs less per call.  Outputs an operator does not produce in some mode
(the last states without `want_last`, dC_initial without `want_dc0`) are empty tensors: an operator returns a fixed
number of tensors.
"""

from __future__ import annotations

from typing import Optional

import torch
from torch import Tensor

from . import _lib

_F32 = torch.float32


def _empty(like: Tensor) -> Tensor:
    return like.new_empty((0,), dtype=_F32)


def _opt(t: Tensor) -> Optional[Tensor]:
    return None if t is None or t.numel() == 0 else t


# ---- chunkwise forward ------------------------------------------------------------------------------------------
@torch.library.custom_op("mlstm_b200::chunkwise_fw", mutates_args=(), device_types="cuda")
def chunkwise_fw(q: Tensor, k: Tensor, v: Tensor, i: Tensor, f: Tensor, c_initial: Optional[Tensor],
                 n_initial: Optional[Tensor], m_initial: Optional[Tensor], chunk_size: int, eps: float, variant: int,
                 impl: str, want_last: bool, keep_states: bool
                 ) -> tuple[Tensor, Tensor, Tensor, Tensor, Tensor, Tensor, Tensor, Tensor]:
    """(H, n_out, m_out, C_states, workspace, C_last, n_last, m_last); `keep_states` only tells the autograd
    registration whether the backward gets the per-chunk states or recomputes them."""
    from .chunkwise import chunkwise_fw_raw, resolve_chunk_size
    L = resolve_chunk_size(q, v, chunk_size, impl)
    out = chunkwise_fw_raw(q, k, v, i, f, c_initial, n_initial, m_initial if variant == _lib.EXP else None,
                           chunk_size=L, eps=eps, variant=variant, impl=impl, want_last=want_last)
    last = (out["C_last"], out["n_last"], out["m_last"]) if want_last else (_empty(q), _empty(q), _empty(q))
    return (out["H"], out["n_out"], out["m_out"], out["C_states"], out["workspace"]) + last


@chunkwise_fw.register_fake
def _(q, k, v, i, f, c_initial, n_initial, m_initial, chunk_size, eps, variant, impl, want_last, keep_states):
    from .chunkwise import resolve_chunk_size
    lib = _lib.load()
    B, NH, S, DHQK = q.shape
    DHHV = v.shape[-1]
    L = resolve_chunk_size(q, v, chunk_size, impl)
    NC = -(-S // L)
    dt, im = _lib.dtype_code(q.dtype), _lib.IMPL[impl]
    sdt = _lib.code_dtype(lib.mlstm_b200_chunkwise_state_dtype(S, DHQK, DHHV, L, dt, im))
    ws = lib.mlstm_b200_chunkwise_workspace_bytes(B, NH, S, DHQK, DHHV, L, dt, variant, im, 0)
    last = ((q.new_empty((B, NH, DHQK, DHHV), dtype=_F32), q.new_empty((B, NH, DHQK), dtype=_F32),
             q.new_empty((B, NH, 1), dtype=_F32)) if want_last else (_empty(q), _empty(q), _empty(q)))
    return (q.new_empty((B, NH, S, DHHV)), q.new_empty((B, NH, S), dtype=_F32), q.new_empty((B, NH, S), dtype=_F32),
            q.new_empty((B, NH, NC + 1, DHQK, DHHV), dtype=sdt), q.new_empty((max(ws, 256),), dtype=torch.uint8)) + last


# ---- chunkwise backward -----------------------------------------------------------------------------------------
@torch.library.custom_op("mlstm_b200::chunkwise_bw", mutates_args=(), device_types="cuda")
def chunkwise_bw(q: Tensor, k: Tensor, v: Tensor, i: Tensor, f: Tensor, m_initial: Optional[Tensor],
                 c_initial: Optional[Tensor], c_states: Optional[Tensor], n_out: Tensor, m_out: Tensor,
                 workspace: Tensor, dh: Tensor, dc_last: Optional[Tensor], chunk_size: int, eps: float, variant: int,
                 impl: str, want_dc0: bool) -> tuple[Tensor, Tensor, Tensor, Tensor, Tensor, Tensor]:
    """(dq, dk, dv, di, df, dc_initial).  c_states = None: the per-chunk states are recomputed (from c_initial)."""
    from .chunkwise import chunkwise_bw_raw, resolve_chunk_size
    L = resolve_chunk_size(q, v, chunk_size, impl)
    dq, dk, dv, di, df, dc0 = chunkwise_bw_raw(
        q, k, v, i, f, m_initial if variant == _lib.EXP else None, c_states, n_out, dh, dc_last, chunk_size=L,
        eps=eps, variant=variant, impl=impl, want_dc_initial=want_dc0, m_out=m_out, fw_workspace=workspace,
        recompute_c_initial=c_initial)
    return dq, dk, dv, di, df, dc0 if want_dc0 else _empty(q)


@chunkwise_bw.register_fake
def _(q, k, v, i, f, m_initial, c_initial, c_states, n_out, m_out, workspace, dh, dc_last, chunk_size, eps, variant,
      impl, want_dc0):
    B, NH, S, DHQK = q.shape
    dc0 = q.new_empty((B, NH, DHQK, v.shape[-1]), dtype=_F32) if want_dc0 else _empty(q)
    return (torch.empty_like(q, memory_format=torch.contiguous_format),
            torch.empty_like(k, memory_format=torch.contiguous_format),
            torch.empty_like(v, memory_format=torch.contiguous_format),
            q.new_empty((B, NH, S), dtype=_F32), q.new_empty((B, NH, S), dtype=_F32), dc0)


def _fw_setup_context(ctx, inputs, output):
    q, k, v, i, f, c_initial, n_initial, m_initial, chunk_size, eps, variant, impl, want_last, keep_states = inputs
    _, n_out, m_out, c_states, workspace = output[:5]
    ctx.cfg = (chunk_size, eps, variant, impl, c_initial is not None, n_initial is not None, m_initial is not None,
               None if c_initial is None else c_initial.dtype, None if n_initial is None else n_initial.dtype,
               (q.shape[0], q.shape[1], q.shape[3]), i.dtype, f.dtype)
    ctx.save_for_backward(q, k, v, i, f, None if keep_states else c_initial, m_initial,
                          c_states if keep_states else None, n_out, m_out, workspace)


def _fw_backward(ctx, dH, _dn_out, _dm_out, _dc_states, _dws, dC_last, _dn_last, _dm_last):
    q, k, v, i, f, c_initial, m_initial, c_states, n_out, m_out, workspace = ctx.saved_tensors
    chunk_size, eps, variant, impl, has_c0, has_n0, has_m0, c0_dtype, n0_dtype, (B, NH, DHQK), i_dtype, f_dtype = ctx.cfg
    if dH is None:
        dH = torch.zeros((B, NH, q.shape[2], v.shape[-1]), dtype=q.dtype, device=q.device)
    dq, dk, dv, di, df, dc0 = chunkwise_bw(q, k, v, i, f, m_initial, c_initial, c_states, n_out, m_out, workspace,
                                          dH.contiguous(), _opt(dC_last), chunk_size, eps, variant, impl, has_c0)
    dn0 = torch.zeros((B, NH, DHQK), dtype=n0_dtype, device=q.device) if has_n0 else None
    dm0 = torch.zeros((B, NH, 1), dtype=m_initial.dtype, device=q.device) if has_m0 else None
    return (dq, dk, dv, di.to(i_dtype), df.to(f_dtype), dc0.to(c0_dtype) if has_c0 else None, dn0, dm0,
            None, None, None, None, None, None)


torch.library.register_autograd("mlstm_b200::chunkwise_fw", _fw_backward, setup_context=_fw_setup_context)


def chunkwise_traced(q, k, v, i, f, c_initial, n_initial, m_initial, return_last_states, eps, chunk_size, impl,
                     recompute_states_in_bw, autocast_kernel_dtype, variant):
    """What the public chunkwise functions do while a trace is being taken: the autocast rule of
    torch.amp.custom_fwd(cast_inputs=...) written out (inside an autocast region floating-point inputs are cast to
    `autocast_kernel_dtype` and the kernel runs with autocast off), then the operator."""
    if torch.is_autocast_enabled("cuda"):
        cast = lambda t: t.to(autocast_kernel_dtype) if (t is not None and t.is_floating_point()) else t  # noqa: E731
        q, k, v, i, f, c_initial, n_initial, m_initial = (cast(t) for t in (q, k, v, i, f, c_initial, n_initial,
                                                                             m_initial))
        with torch.autocast("cuda", enabled=False):
            out = chunkwise_fw(q, k, v, i, f, c_initial, n_initial, m_initial, chunk_size, eps, variant, impl,
                               return_last_states, not recompute_states_in_bw)
    else:
        out = chunkwise_fw(q, k, v, i, f, c_initial, n_initial, m_initial, chunk_size, eps, variant, impl,
                           return_last_states, not recompute_states_in_bw)
    return out[0], out[5], out[6], out[7]


# ---- decode -----------------------------------------------------------------------------------------------------
@torch.library.custom_op("mlstm_b200::step", mutates_args=(), device_types="cuda")
def step(q: Tensor, k: Tensor, v: Tensor, i: Tensor, f: Tensor, c: Tensor, n: Tensor, m: Tensor, eps: float,
         state_is_bf16: bool) -> tuple[Tensor, Tensor, Tensor, Tensor]:
    from .recurrent import mlstm_recurrent_step__b200_fw
    h, (c_new, n_new, m_new) = mlstm_recurrent_step__b200_fw(
        c, n, m, q, k, v, i, f, eps=eps, dtype_state=torch.bfloat16 if state_is_bf16 else _F32)
    return h, c_new, n_new, m_new


@step.register_fake
def _(q, k, v, i, f, c, n, m, eps, state_is_bf16):
    sdt = torch.bfloat16 if state_is_bf16 else _F32
    return (torch.empty_like(v, memory_format=torch.contiguous_format), c.new_empty(c.shape, dtype=sdt),
            n.new_empty(n.shape, dtype=sdt), m.new_empty(m.shape, dtype=sdt))


@torch.library.custom_op("mlstm_b200::step_sequence", mutates_args=(), device_types="cuda")
def step_sequence(q: Tensor, k: Tensor, v: Tensor, i: Tensor, f: Tensor, c_initial: Optional[Tensor],
                  n_initial: Optional[Tensor], m_initial: Optional[Tensor], eps: float
                  ) -> tuple[Tensor, Tensor, Tensor, Tensor]:
    from .recurrent import mlstm_recurrent_sequence__b200
    h, (c_new, n_new, m_new) = mlstm_recurrent_sequence__b200(q, k, v, i, f, c_initial, n_initial, m_initial,
                                                              return_last_states=True, eps=eps)
    return h, c_new, n_new, m_new


@step_sequence.register_fake
def _(q, k, v, i, f, c_initial, n_initial, m_initial, eps):
    B, NH, S, DHQK = q.shape
    DHHV = v.shape[-1]
    return (torch.empty_like(v, memory_format=torch.contiguous_format), q.new_empty((B, NH, DHQK, DHHV), dtype=_F32),
            q.new_empty((B, NH, DHQK), dtype=_F32), q.new_empty((B, NH, 1), dtype=_F32))


# ---- the operators around a recurrence ----------------------------------------------------------------------------
# (their checks of arguments are the native host module's, made when an operator runs)
def _contig(t: Tensor) -> Tensor:
    return torch.empty_like(t, memory_format=torch.contiguous_format)


@torch.library.custom_op("mlstm_b200::layer_norm", mutates_args=(), device_types="cuda")
def layer_norm(x: Tensor, weight: Optional[Tensor], bias: Optional[Tensor], eps: float) -> tuple[Tensor, Tensor, Tensor]:
    """(y, mean, rstd)"""
    return _lib.host().layer_norm_fw(x, weight, bias, eps)


@layer_norm.register_fake
def _(x, weight, bias, eps):
    rows = 1
    for n in x.shape[:-1]:
        rows = rows * n
    return _contig(x), x.new_empty((rows,), dtype=_F32), x.new_empty((rows,), dtype=_F32)


@torch.library.custom_op("mlstm_b200::layer_norm_bw", mutates_args=(), device_types="cuda")
def layer_norm_bw(x: Tensor, weight: Optional[Tensor], mean: Tensor, rstd: Tensor, dy: Tensor, heads: bool,
                  param_dtype: torch.dtype) -> tuple[Tensor, Tensor, Tensor]:
    """dx lies as torch.empty_like(x) does, which for an x that covers its memory once is where the kernels write it."""
    dx, dw, db = _lib.host().layer_norm_bw(x, weight, mean, rstd, dy, heads, param_dtype, True, True)
    if dx.stride() != x.stride():   # (x in parts of wider rows, or without memory of its own)
        like = torch.empty_like(x)
        dx = dx if dx.stride() == like.stride() else like.copy_(dx)
    return dx, dw, db


@layer_norm_bw.register_fake
def _(x, weight, mean, rstd, dy, heads, param_dtype):
    p = x.new_empty(x.shape[-2:] if heads else x.shape[-1:], dtype=param_dtype)
    return torch.empty_like(x), p, torch.empty_like(p)


def _norm_setup_context(ctx, inputs, output):
    x, weight, bias, _ = inputs
    p = weight if weight is not None else bias
    ctx.save_for_backward(x, weight, output[1], output[2])
    ctx.cfg = (p is not None and p.dim() == 2, _F32 if p is None else p.dtype, weight is not None, bias is not None)


def _norm_backward(ctx, dy, _dmean, _drstd):
    x, weight, mean, rstd = ctx.saved_tensors
    heads, pdt, has_w, has_b = ctx.cfg
    dx, dw, db = layer_norm_bw(x, weight, mean, rstd, dy, heads, pdt)
    return dx, dw if has_w else None, db if has_b else None, None


torch.library.register_autograd("mlstm_b200::layer_norm", _norm_backward, setup_context=_norm_setup_context)


@torch.library.custom_op("mlstm_b200::short_conv", mutates_args=(), device_types="cuda")
def short_conv(x: Tensor, weight: Tensor, bias: Optional[Tensor], x_initial: Optional[Tensor], want_last: bool, silu: bool
               ) -> tuple[Tensor, Tensor]:
    y, last = _lib.host().short_conv(x, weight, bias, x_initial, want_last, silu)
    return y, last if want_last else x.new_empty((0,))


@short_conv.register_fake
def _(x, weight, bias, x_initial, want_last, silu):
    return _contig(x), x.new_empty((x.shape[0], weight.shape[1] - 1, x.shape[2]) if want_last else (0,))


@torch.library.custom_op("mlstm_b200::short_conv_bw", mutates_args=(), device_types="cuda")
def short_conv_bw(x: Tensor, weight: Tensor, bias: Optional[Tensor], x_initial: Optional[Tensor], dy: Optional[Tensor],
                  dlast: Optional[Tensor], silu: bool) -> tuple[Tensor, Tensor, Tensor, Tensor]:
    dx, dw, db, d0 = _lib.host().short_conv_bw(x, weight, bias, x_initial, dy, dlast, silu, True, bias is not None,
                                               x_initial is not None)
    none = x.new_empty((0,))
    return dx, dw, none if db is None else db, none.clone() if d0 is None else d0


@short_conv_bw.register_fake
def _(x, weight, bias, x_initial, dy, dlast, silu):
    return (_contig(x), _contig(weight), x.new_empty((0,)) if bias is None else _contig(bias),
            x.new_empty((0,)) if x_initial is None else _contig(x_initial))


def _conv_setup_context(ctx, inputs, output):
    x, weight, bias, x_initial, want_last, silu = inputs
    ctx.save_for_backward(x, weight, bias, x_initial)
    ctx.cfg = (want_last, silu)


def _conv_backward(ctx, dy, dlast):
    x, weight, bias, x_initial = ctx.saved_tensors
    want_last, silu = ctx.cfg
    dx, dw, db, d0 = short_conv_bw(x, weight, bias, x_initial, dy, dlast if want_last else None, silu)
    return dx, dw, None if bias is None else db, None if x_initial is None else d0, None, None


torch.library.register_autograd("mlstm_b200::short_conv", _conv_backward, setup_context=_conv_setup_context)


@torch.library.custom_op("mlstm_b200::short_conv_step", mutates_args=(), device_types="cuda")
def short_conv_step(x: Tensor, state: Tensor, weight: Tensor, bias: Optional[Tensor], silu: bool) -> tuple[Tensor, Tensor]:
    return _lib.host().short_conv_step(x, state, weight, bias, silu, None)


@short_conv_step.register_fake
def _(x, state, weight, bias, silu):
    return _contig(x), _contig(state)


@torch.library.custom_op("mlstm_b200::short_conv_step_into", mutates_args=("state_new",), device_types="cuda")
def short_conv_step_into(x: Tensor, state: Tensor, weight: Tensor, bias: Optional[Tensor], silu: bool, state_new: Tensor) -> Tensor:
    return _lib.host().short_conv_step(x, state, weight, bias, silu, state_new)[0]


@short_conv_step_into.register_fake
def _(x, state, weight, bias, silu, state_new):
    return _contig(x)


@torch.library.custom_op("mlstm_b200::ssm_scan", mutates_args=(), device_types="cuda")
def ssm_scan(x: Tensor, dt: Tensor, a: Tensor, b: Tensor, c: Tensor, skip: Optional[Tensor], z: Optional[Tensor],
             dt_bias: Optional[Tensor], softplus: bool, h_initial: Optional[Tensor], keep: bool = True, want_last: bool = True
             ) -> tuple[Tensor, Tensor, Tensor]:
    """(y, h_last, checkpoints); without `keep` no checkpoints, and no gradient"""
    y, last, checkpoints = _lib.host().ssm_scan_fw(x, dt, a, b, c, skip, z, dt_bias, h_initial, softplus, keep, want_last)
    return y, last if want_last else _empty(x), checkpoints if keep else x.new_empty((0,), dtype=torch.uint8)


@ssm_scan.register_fake
def _(x, dt, a, b, c, skip, z, dt_bias, softplus, h_initial, keep=True, want_last=True):
    B, S, D = x.shape
    N = a.shape[1]
    # (worked out here, not asked for: S may be a symbol; sixteen tokens to a checkpoint)
    n = torch.sym_max(B * ((S + 15) // 16) * D * _lib.load().mlstm_b200_ssm_checkpoint_bytes(1, 1, 1, int(N)), 256) if keep else 0
    return (_contig(x), x.new_empty((B, D, N) if want_last else (0,), dtype=_F32), x.new_empty((n,), dtype=torch.uint8))


@torch.library.custom_op("mlstm_b200::ssm_scan_bw", mutates_args=(), device_types="cuda")
def ssm_scan_bw(x: Tensor, dt: Tensor, a: Tensor, b: Tensor, c: Tensor, skip: Optional[Tensor], z: Optional[Tensor],
                dt_bias: Optional[Tensor], softplus: bool, h_initial: Optional[Tensor], checkpoints: Tensor,
                dy: Optional[Tensor], dh_last: Optional[Tensor]
                ) -> tuple[Tensor, Tensor, Tensor, Tensor, Tensor, Tensor, Tensor, Tensor, Tensor]:
    g = _lib.host().ssm_scan_bw(x, dt, a, b, c, skip, z, dt_bias, h_initial, softplus, checkpoints, dy, dh_last)
    return tuple(x.new_empty((0,)) if t is None else t for t in g)


@ssm_scan_bw.register_fake
def _(x, dt, a, b, c, skip, z, dt_bias, softplus, h_initial, checkpoints, dy, dh_last):
    like = lambda t: x.new_empty((0,)) if t is None else _contig(t)  # noqa: E731
    return tuple(like(t) for t in (x, dt, a, b, c, skip, z, dt_bias, h_initial))


def _ssm_setup_context(ctx, inputs, output):
    x, dt, a, b, c, skip, z, dt_bias, softplus, h_initial, keep, want_last = inputs
    ctx.save_for_backward(x, dt, a, b, c, skip, z, dt_bias, h_initial, output[2])
    ctx.cfg = (softplus, keep, want_last)


def _ssm_backward(ctx, dy, dh_last, _dck):
    x, dt, a, b, c, skip, z, dt_bias, h_initial, checkpoints = ctx.saved_tensors
    softplus, keep, want_last = ctx.cfg
    if not keep:
        raise RuntimeError("mlstm_b200::ssm_scan: no gradient without checkpoints (keep=False)")
    dx, ddt, da, db, dc, dskip, dz, dbias, dh0 = ssm_scan_bw(x, dt, a, b, c, skip, z, dt_bias, softplus, h_initial,
                                                             checkpoints, dy, dh_last if want_last else None)
    return (dx, ddt, da, db, dc, None if skip is None else dskip, None if z is None else dz, None if dt_bias is None else dbias,
            None, None if h_initial is None else dh0, None, None)


torch.library.register_autograd("mlstm_b200::ssm_scan", _ssm_backward, setup_context=_ssm_setup_context)


@torch.library.custom_op("mlstm_b200::ssm_step", mutates_args=(), device_types="cuda")
def ssm_step(x: Tensor, dt: Tensor, a: Tensor, b: Tensor, c: Tensor, h: Tensor, skip: Optional[Tensor], z: Optional[Tensor],
             dt_bias: Optional[Tensor], softplus: bool) -> tuple[Tensor, Tensor]:
    return _lib.host().ssm_step(x, dt, a, b, c, skip, z, dt_bias, h, softplus, None)


@ssm_step.register_fake
def _(x, dt, a, b, c, h, skip, z, dt_bias, softplus):
    return _contig(x), h.new_empty(h.shape, dtype=_F32)


@torch.library.custom_op("mlstm_b200::ssm_step_into", mutates_args=("h_new",), device_types="cuda")
def ssm_step_into(x: Tensor, dt: Tensor, a: Tensor, b: Tensor, c: Tensor, h: Tensor, skip: Optional[Tensor], z: Optional[Tensor],
                  dt_bias: Optional[Tensor], softplus: bool, h_new: Tensor) -> Tensor:
    return _lib.host().ssm_step(x, dt, a, b, c, skip, z, dt_bias, h, softplus, h_new)[0]


@ssm_step_into.register_fake
def _(x, dt, a, b, c, h, skip, z, dt_bias, softplus, h_new):
    return _contig(x)
