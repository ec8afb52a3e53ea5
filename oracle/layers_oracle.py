"""numpy restatement (float64) of the operators around a recurrence: layer norm, short causal convolution, selective state space
scan, with their gradients written out.

Every function returns {name: (value, error)}: `error` bounds, in units of 2^-24, what f32 arithmetic in any order of the sums may be
off by, to first order: each rounding of a value adds one unit of the sum of the absolute terms behind it, an exponential, a
logarithm and a division a few, and an exponential passes the error of its argument on times itself: e^x as 2^(x log2 e) with both
the constant and the product rounded is off by 2 |x| units of itself (log2 e is 1.44269504 +- 2^-26, half a unit of 1.44 |x|, and the
product half a step, at most one unit of it; times ln 2 that is 1.5 |x|) and 4 more (2^x off by 2^-22).  Rounding of a result to its
element type comes on top (half a step).  The constants are counts of such roundings, rounded up."""

from __future__ import annotations

import numpy as np


def _sigmoid(v):
    return 0.5 * (1 + np.tanh(0.5 * v))


# ---- layer norm -----------------------------------------------------------------------------------------------------
# Sums over D: at most 16 in a thread and 10 across lanes and warps, so 32 units cover a mean; 64 the variance and its root too.
def layer_norm(x, weight=None, bias=None, eps=1e-6, dy=None):
    w = np.ones(x.shape[-1]) if weight is None else weight
    b = np.zeros_like(w) if bias is None else bias
    mu = x.mean(-1, keepdims=True)
    var = ((x - mu) ** 2).mean(-1, keepdims=True)
    rstd = 1 / np.sqrt(var + eps)
    n = (x - mu) * rstd
    centred = (np.abs(x) + np.abs(x).mean(-1, keepdims=True)) * rstd   # what a rounding of x - mu is relative to
    # an error of the mean shifts every x - mu, and enters the variance in the second order and through their sum (zero)
    n_err = 64 * centred + 64 * np.abs(n)
    r = {"y": (n * w + b, n_err * np.abs(w) + 4 * (np.abs(n * w) + np.abs(b)))}
    if dy is None:
        return r
    g = dy * w
    c1, c2 = g.mean(-1, keepdims=True), (g * n).mean(-1, keepdims=True)
    ag = np.abs(g)
    c1_err = 34 * ag.mean(-1, keepdims=True)
    c2_err = (ag * (n_err + 36 * np.abs(n))).mean(-1, keepdims=True)
    dx_err = c1_err + 4 * np.abs(c1) + np.abs(n) * c2_err + np.abs(c2) * n_err + 4 * np.abs(n * c2) + 4 * ag
    r["dx"] = (rstd * (g - c1 - n * c2), rstd * (dx_err + 72 * (ag + np.abs(c1) + np.abs(n * c2))))
    axes = tuple(range(x.ndim - w.ndim))
    rows = int(np.prod([x.shape[i] for i in axes], dtype=np.int64))
    r["dweight"] = ((dy * n).sum(axes), (np.abs(dy) * (n_err + (rows + 32) * np.abs(n))).sum(axes))
    r["dbias"] = (dy.sum(axes), (rows + 32) * np.abs(dy).sum(axes))
    return r


# ---- short convolution ----------------------------------------------------------------------------------------------
def short_conv(x, weight, bias=None, x_initial=None, silu=False, dy=None, dlast=None):
    (B, S, D), W = x.shape, weight.shape[1]
    v = np.zeros((B, S + W - 1, D))
    v[:, W - 1:] = x
    if x_initial is not None:
        v[:, :W - 1] = x_initial
    u = np.zeros((B, S, D)) + (0 if bias is None else bias)
    mag = np.abs(u)
    for j in range(W):
        u = u + weight[:, j] * v[:, j:j + S]
        mag = mag + np.abs(weight[:, j] * v[:, j:j + S])
    u_err = 6 * mag
    s = _sigmoid(u)
    # sigmoid and its product: 8 units, and 2 |u| (1 - s) from the exponential; the derivative of u sigmoid(u) is below 1.1
    se = 2 * np.abs(u) * (1 - s)
    r = {"y": (u * s, 1.1 * u_err + (8 + se) * np.abs(u * s)) if silu else (u, u_err), "last": (v[:, S:], np.zeros((B, W - 1, D)))}
    if dy is None:
        return r
    if silu:   # the second derivative of u sigmoid(u) is below 0.6
        f = s * (1 + u * (1 - s))
        # (an error of s also moves 1 - s: by at most as many units of s)
        k, k_err = dy * f, np.abs(dy) * (0.6 * u_err + (16 + se) * s * (1 + np.abs(u)))
    else:
        k, k_err = dy, np.zeros_like(dy)
    dv, dv_err = np.zeros_like(v), np.zeros_like(v)
    if dlast is not None:
        dv[:, S:] += dlast
        dv_err[:, S:] += 2 * np.abs(dlast)
    dw, dw_err = np.zeros((D, W)), np.zeros((D, W))
    n = B * S + 32
    for j in range(W):
        dv[:, j:j + S] += weight[:, j] * k
        dv_err[:, j:j + S] += np.abs(weight[:, j]) * (k_err + 8 * np.abs(k))
        dw[:, j] = (k * v[:, j:j + S]).sum((0, 1))
        dw_err[:, j] = (np.abs(v[:, j:j + S]) * (k_err + n * np.abs(k))).sum((0, 1))
    r.update(dx=(dv[:, W - 1:], dv_err[:, W - 1:]), dx_initial=(dv[:, :W - 1], dv_err[:, :W - 1]), dweight=(dw, dw_err),
             dbias=(k.sum((0, 1)), (k_err + n * np.abs(k)).sum((0, 1))))
    return r


# ---- selective state space scan -------------------------------------------------------------------------------------
def ssm_scan(x, dt, a, b, c, skip=None, z=None, dt_bias=None, softplus=False, h_initial=None, dy=None, dh_last=None, summed=0):
    """`summed`: the most steps whose sum the kernels may take the exponential of (a segment's decay)."""
    B, S, D = x.shape
    N = a.shape[1]
    flat = b.ndim == 3
    b4, c4 = (b[:, :, None], c[:, :, None]) if flat else (b, c)
    G = b4.shape[2]
    bd, cd = np.repeat(b4, D // G, 2), np.repeat(c4, D // G, 2)          # (B, S, D, N)
    skip_ = np.zeros(D) if skip is None else skip
    raw = dt + (0 if dt_bias is None else dt_bias)
    step = np.logaddexp(raw, 0) if softplus else raw
    # the step: 12 units of itself (softplus), and what the rounding of dt + dt_bias and the exponential's argument do to it: |raw|
    # and 2 |raw| units, as the derivative of softplus is at most itself; the argument of an exponential has three more
    rel = 12 + np.maximum(1, 3 * np.abs(raw))
    arg = step[..., None] * a
    dec = np.exp(arg)
    arg_err = np.abs(arg) * (rel[..., None] + 3 + summed)
    inc = (step * x)[..., None] * bd
    h = np.zeros((B, D, N)) if h_initial is None else h_initial.astype(np.float64)
    H, e = np.abs(h), np.zeros((B, D, N))
    hs, Hs, es = [h], [H], [e]
    for t in range(S):
        through = dec[:, t] * H
        e = dec[:, t] * e + (arg_err[:, t] + 6) * through + (rel[:, t, :, None] + 4) * np.abs(inc[:, t])
        h, H = dec[:, t] * h + inc[:, t], through + np.abs(inc[:, t])
        hs.append(h), Hs.append(H), es.append(e)
    hs, Hs, es = (np.stack(v, 1) for v in (hs, Hs, es))                     # (B, S + 1, D, N)
    out = (hs[:, 1:] * cd).sum(-1) + skip_ * x
    O = (Hs[:, 1:] * np.abs(cd)).sum(-1) + np.abs(skip_ * x)
    o_err = (es[:, 1:] * np.abs(cd)).sum(-1) + 16 * O
    if z is None:
        s, sz, dsz, gate_err = np.ones_like(x), np.ones_like(x), np.zeros_like(x), np.zeros_like(x)
    else:
        s = _sigmoid(z)
        sz, dsz = z * s, s * (1 + z * (1 - s))
        gate_err = 12 + 2 * np.abs(z) * (1 - s)   # units of s and of z s
    r = {"y": (out * sz, np.abs(sz) * (o_err + gate_err * O)), "h_last": (hs[:, S], es[:, S] + Hs[:, S])}
    if dy is None:
        return r
    dout = dy * sz
    Dm = np.abs(dout)
    d_err = gate_err * Dm
    q = np.zeros((B, D, N)) if dh_last is None else dh_last.astype(np.float64)   # e_{t+1} g_{t+1}
    Q, qe = np.abs(q), np.zeros((B, D, N))
    g, Gm, ge = (np.zeros((B, S, D, N)) for _ in range(3))
    for t in range(S - 1, -1, -1):
        ac = np.abs(cd[:, t])
        g[:, t], Gm[:, t] = dout[:, t, :, None] * cd[:, t] + q, Dm[:, t, :, None] * ac + Q
        ge[:, t] = d_err[:, t, :, None] * ac + qe + 2 * Gm[:, t]
        q, Q = dec[:, t] * g[:, t], dec[:, t] * Gm[:, t]
        qe = dec[:, t] * ge[:, t] + (arg_err[:, t] + 6) * Q
    gb, GB = (g * bd).sum(-1), (Gm * np.abs(bd)).sum(-1)
    gb_err = (ge * np.abs(bd)).sum(-1) + 16 * GB
    T = g * dec * hs[:, :-1]
    Tm = Gm * dec * Hs[:, :-1]
    Te = dec * (ge * Hs[:, :-1] + Gm * es[:, :-1]) + (arg_err + 10) * Tm
    st = np.abs(step)
    r["dx"] = (step * gb + skip_ * dout, st * (gb_err + (rel + 4) * GB) + np.abs(skip_) * (d_err + 4 * Dm))
    dr = (T * a).sum(-1) + x * gb
    Dr = (Tm * np.abs(a)).sum(-1) + np.abs(x) * GB
    dr_err = (Te * np.abs(a)).sum(-1) + np.abs(x) * gb_err + 20 * Dr
    if softplus:   # the logistic function's own error: 6 units, and that of its argument
        sg = _sigmoid(raw)
        dr, dr_err, Dr = dr * sg, dr_err * sg + Dr * sg * (8 + 3 * np.abs(raw)), Dr * sg
    r["ddt"] = (dr, dr_err)
    n = S + B + 32
    by = lambda v: v.reshape(B, S, G, D // G, N).sum(3).reshape(b.shape)  # noqa: E731
    dn = D // G + 16
    sx = (step * x)[..., None]
    r["db"] = (by(g * sx), by(np.abs(sx) * (ge + (rel[..., None] + dn) * Gm)))
    r["dc"] = (by(hs[:, 1:] * dout[..., None]), by(Dm[..., None] * (es[:, 1:] + dn * Hs[:, 1:]) + d_err[..., None] * Hs[:, 1:]))
    r["da"] = ((T * step[..., None]).sum((0, 1)), (st[..., None] * (Te + (rel[..., None] + n) * Tm)).sum((0, 1)))
    r["ddt_bias"] = (dr.sum((0, 1)), (dr_err + n * Dr).sum((0, 1)))
    r["dskip"] = ((dout * x).sum((0, 1)), (np.abs(x) * (d_err + n * Dm)).sum((0, 1)))
    r["dh_initial"] = (q, qe)
    if z is not None:
        r["dz"] = (dy * out * dsz, np.abs(dy) * (1.1 * (o_err + 8 * O) + (16 + gate_err) * O * s * (1 + np.abs(z))))
    return r
