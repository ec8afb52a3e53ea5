"""numpy restatement (float64) of the gated linear recurrence, with its gradients written out, and of the counter-based generator and
the dropout by it.

As in layers_oracle.py, results are {name: (value, error)}, the error in units of 2^-24 of what f32 arithmetic in any order of the
joins may be off by, to first order.  What the gates add (derivations beside them): e^-v is off by E = 2 |v| + 4 units of itself; a sum, a
product, a reciprocal and a root by 1, 1, 2 and 3."""

from __future__ import annotations

import numpy as np


def _logistic(v):
    """sigmoid(v), 1 - sigmoid(v), and the units of both."""
    s, c = 1 / (1 + np.exp(-v)), 1 / (1 + np.exp(v))
    E = 2 * np.minimum(np.abs(v), 1e3) + 4   # (beyond, e^-v is zero or infinite, and exact)
    # v <= 0: s = 1 / (1 + e) moves by c E, and 3; c = 1 - s by s / c <= 1 of that, and 1.  v > 0: c = e / (1 + e) moves by s E, and 4;
    # s = 1 - c by c / s of that, and 1
    with np.errstate(divide="ignore", over="ignore"):
        s_err = np.where(v > 0, c * E + 4 * c / s + 1, c * E + 3)
        c_err = np.where(v > 0, s * E + 4, s * E + 3 * np.minimum(1, s / c) + 1)
    return s, c, s_err, c_err


def gated_scan(x, f, i=None, z=None, rate=None, h_initial=None, input_scale=None, dy=None, dh_last=None):
    B, S, D = x.shape
    sf, cf, sf_err, cf_err = _logistic(f)
    if rate is None:
        a, rest, a_err, rest_err = sf, cf, sf_err, cf_err
    else:
        rho = -rate * sf
        a, rest = np.exp(-rho), -np.expm1(-rho)
        rho_err = sf_err + 1
        # below 1/2: rho times a polynomial, d log(rest) <= d log(rho); one minus it.  Else an exponential; one minus it
        near = (rho < 0.5) & (rho >= 0)
        safe = np.where(near, 1, rest)
        a_err = np.where(near, rest / a * (rho_err + 4) + 1, np.abs(rho) * (rho_err + 2) + 4)
        rest_err = np.where(near, rho_err + 4, np.abs(a / safe) * a_err + 1)
    rest2 = rest * (1 + a)
    rest2_err = rest_err + a_err + 1
    if input_scale is None:
        s, s_err = np.ones_like(a), np.zeros_like(a)
    elif input_scale == "convex":
        s, s_err = rest, rest_err
    else:
        s, s_err = np.sqrt(rest2), rest2_err / 2 + 4
    g, cg, g_err, cg_err = (np.ones_like(x), np.zeros_like(x), np.zeros_like(x), np.zeros_like(x)) if i is None else _logistic(i)
    gx = g * x
    gx_err = g_err + 1
    u = s * gx
    u_err = s_err + gx_err + 1
    h = np.zeros((B, D)) if h_initial is None else h_initial.astype(np.float64)
    H, e = np.abs(h), np.zeros((B, D))
    hs, Hs, es = [h], [H], [e]
    for t in range(S):
        # a token's factor is rounded into the product of its run, the product's product with what came before is, and their sums are
        e = a[:, t] * e + (a_err[:, t] + 4) * a[:, t] * H + (u_err[:, t] + 4) * np.abs(u[:, t])
        h, H = a[:, t] * h + u[:, t], a[:, t] * H + np.abs(u[:, t])
        hs.append(h), Hs.append(H), es.append(e)
    hs, Hs, es = (np.stack(v, 1) for v in (hs, Hs, es))
    if z is None:
        sz, o, o_err = np.ones_like(x), np.ones_like(x), np.zeros_like(x)
    else:
        sz, cz, sz_err, cz_err = _logistic(z)
        o, o_err = z * sz, sz_err + 1
    now, Now, now_err = hs[:, 1:], Hs[:, 1:], es[:, 1:]
    r = {"y": (now * o, np.abs(o) * (now_err + (o_err + 1) * Now)), "h_last": (hs[:, S], es[:, S])}
    if dy is None:
        return r
    q = np.zeros((B, D)) if dh_last is None else dh_last.astype(np.float64)   # a_{t+1} G_{t+1}
    Q, qe = np.abs(q), np.zeros((B, D))
    G, Gm, Ge = (np.zeros((B, S, D)) for _ in range(3))
    for t in range(S - 1, -1, -1):
        d = dy[:, t] * o[:, t]
        G[:, t], Gm[:, t] = d + q, np.abs(d) + Q
        Ge[:, t] = qe + (o_err[:, t] + 5) * np.abs(d)
        q, Q = a[:, t] * G[:, t], a[:, t] * Gm[:, t]
        qe = a[:, t] * Ge[:, t] + (a_err[:, t] + 4) * Q
    r["dh_initial"] = (q, qe)
    r["dx"] = (G * s * g, s * g * (Ge + (s_err + g_err + 3) * Gm))
    if i is not None:
        r["di"] = (G * u * cg, np.abs(u * cg) * (Ge + (u_err + cg_err + 3) * Gm))
    if z is not None:
        k = sz * (1 + z * cz)
        # z (1 - sigmoid) and one plus it: units of 1 + |z| (1 - sigmoid)
        k_err = sz * ((cz_err + 2) * np.abs(z) * cz + (sz_err + 2) * (1 + np.abs(z) * cz))
        r["dz"] = (dy * now * k, np.abs(dy) * (np.abs(k) * (now_err + 3 * Now) + k_err * Now))
    # through a: the state before, and what the scale does to the input
    if input_scale is None:
        back, back_err = np.zeros_like(x), np.zeros_like(x)
    elif input_scale == "convex":
        back, back_err = gx, gx_err * np.abs(gx)
    else:
        # a sigmoid(i) x / s, finite where s is zero: what it is multiplied by is zero too
        inv = 1 / np.sqrt(np.maximum(rest2, 2.0 ** -126))
        back = a * gx * inv
        back_err = np.abs(back) * (a_err + gx_err + rest2_err / 2 + 5)
    w = hs[:, :-1] - back
    W = Hs[:, :-1] + np.abs(back)
    w_err = es[:, :-1] + back_err + W
    ga = a * G
    v, V, v_err = ga * w, a * Gm * W, a * (Ge * W + Gm * w_err + (a_err + 3) * Gm * W)
    if rate is None:
        r["df"] = (v * rest, rest * (v_err + (rest_err + 2) * V))
    else:
        m = np.abs(rate) * sf * cf
        r["df"] = (v * rate * sf * cf, m * (v_err + (sf_err + cf_err + 4) * V))
        # sums over tokens and sequences: at most as many roundings behind a term as there are terms
        r["drate"] = ((v * sf).sum((0, 1)), (sf * (v_err + (sf_err + 2 + S * B + 32) * V)).sum((0, 1)))
    return r


# ---- what a state forgets --------------------------------------------------------------------------------------------
# Tokens of one factor a = exp(-rho).  f32 holds a to 2^-25 and products of joined runs to 2^-24 of themselves, about one to a token
# (seven to a run of eight, some to a unit of runs): 2^-23 a token with half of that to spare; rho has 2^-20 of itself (_logistic, a
# product and a polynomial).
def kept_state(S, rho):
    """What S tokens without input leave of a state of one: 1 - it, and by how much of itself that may be off."""
    gone = -np.expm1(-S * rho)
    return gone, S * (2.0 ** -23 + rho * 2.0 ** -20) / gone


def constant_input(S, rho):
    """The "convex" state after S inputs of one: its value, and by how much of itself it may be off: a token's input (2^-20), and for
    each token that is remembered its factor and the sums, which round as often as the products."""
    return -np.expm1(-S * rho), np.minimum(S, 1 / rho) * 2.0 ** -22 + 2.0 ** -19


# ---- the generator --------------------------------------------------------------------------------------------------
def philox4x32(counter, key, rounds):
    """Salmon, Moraes, Dror, Shaw, Parallel random numbers: as easy as 1, 2, 3 (2011).  counter (..., 4), key (2): 32-bit words."""
    mask = np.uint64(0xFFFFFFFF)
    c = [np.asarray(counter)[..., k].astype(np.uint64) for k in range(4)]
    k0, k1 = (int(k) for k in key)
    for _ in range(rounds):
        p0, p1 = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        c = [(p1 >> np.uint64(32)) ^ c[1] ^ np.uint64(k0), p1 & mask, (p0 >> np.uint64(32)) ^ c[3] ^ np.uint64(k1), p0 & mask]
        k0, k1 = (k0 + 0x9E3779B9) & 0xFFFFFFFF, (k1 + 0xBB67AE85) & 0xFFFFFFFF
    return np.stack(c, -1)


def kept(shape, p, seed, offset=0, first=0):
    """Which elements of a tensor of this shape dropout keeps; `first`: the index of its first element."""
    n = int(np.prod(shape, dtype=np.int64))
    quads = np.arange(first // 4, (first + n + 3) // 4, dtype=np.uint64)
    lo = np.uint64(0xFFFFFFFF)
    ctr = np.stack([quads & lo, quads >> np.uint64(32), np.full_like(quads, offset & 0xFFFFFFFF), np.full_like(quads, offset >> 32)], -1)
    words = philox4x32(ctr, (seed & 0xFFFFFFFF, seed >> 32), 7).reshape(-1)[first % 4:first % 4 + n]
    return (words >= round(p * 2.0 ** 32)).reshape(shape)


def dropout(x, p, seed, offset=0, residual=None, dy=None):
    keep = kept(x.shape, p, seed, offset)
    scale = 1 / (1 - p) if round(p * 2.0 ** 32) < 2 ** 32 else 0.0
    v = np.where(keep, x * scale, 0.0)
    r = {"y": (v, 2 * np.abs(v)) if residual is None else (residual + v, 3 * np.abs(v) + np.abs(residual))}
    if dy is not None:
        d = np.where(keep, dy * scale, 0.0)
        r["dx"] = (d, 2 * np.abs(d))
        r["dresidual"] = (dy, np.zeros_like(dy))
    return r
