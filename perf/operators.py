"""The operators of a recurrent layer around its recurrence, as cases that can be timed and compared: layer norm, the short
causal convolution, and the selective state space scan with its step for single tokens.

Where `own` is false, run() computes them from elementary torch operations; where it is true, through this package.

  norm        y = (x - mean) / sqrt(var + eps) * weight + bias over the last axis; with heads, x is the (B, NH, S, DH) output of a
              recurrence, seen as (B, S, NH, DH), and weight and bias are (NH, DH)
  conv        y_t = act(bias + sum_j weight_j x_{t-W+1+j}) per channel, over x (B, S, D); conv_step is one token of it
  ssm         dt' = softplus(dt + dt_bias); h_t = exp(dt'_t a) h_{t-1} + dt'_t x_t b_t; y_t = (c_t . h_t + skip x_t) silu(z_t)
              over x, dt, z (B, S, D), b, c (B, S, G, N) and a state (B, D, N); ssm_step is one token of it
"""

import math

import torch

own = False

_DTYPE = {"bf16": torch.bfloat16, "fp16": torch.float16, "f32": torch.float32}
_BYTES = {"bf16": 2, "fp16": 2, "f32": 4}
_EPS = 1e-5


def listed():
    return [
        # the norm of one generated token of four users: the smallest call, launch latency and host time count
        dict(name="norm_decode", kind="norm", train=False, B=4, S=1, NH=1, D=4096, heads=False, dtype="bf16", param="bf16"),
        # the norm in front of a layer while a prompt of any length is read
        dict(name="norm_prefill_fp16", kind="norm", train=False, B=1, S=8077, NH=1, D=4096, heads=False, dtype="fp16",
             param="f32"),
        # the norm of the heads behind a recurrence in a training step: 32 768 tokens, read from (B, NH, S, DH) in place
        dict(name="norm_heads_train", kind="norm", train=True, B=8, S=4096, NH=16, D=256, heads=True, dtype="bf16", param="f32"),
        # a small model in single precision whose width is no multiple of anything
        dict(name="norm_train_f32", kind="norm", train=True, B=3, S=777, NH=1, D=1001, heads=False, dtype="f32", param="f32"),
        # one token of sixteen users
        dict(name="conv_decode", kind="conv_step", B=16, D=4096, W=4, act=True, dtype="bf16"),
        # a batch of long prompts, the last tokens kept for the decode that follows
        dict(name="conv_prefill", kind="conv", train=False, B=4, S=8077, D=2048, W=4, act=True, init=False, dtype="bf16"),
        # a training step of one layer
        dict(name="conv_train", kind="conv", train=True, B=8, S=4096, D=2048, W=4, act=True, init=False, dtype="bf16"),
        # segments of longer texts in single precision: three taps, odd sizes, the tokens before given
        dict(name="conv_train_f32", kind="conv", train=True, B=3, S=777, D=1001, W=3, act=False, init=True, dtype="f32"),
        # one token of a serving batch: 33 MB of states in and out
        dict(name="ssm_decode", kind="ssm_step", B=64, D=4096, N=16, G=1, dtype="bf16"),
        # one long document
        dict(name="ssm_prefill_long", kind="ssm", train=False, B=1, S=16384, D=2048, N=16, G=1, gate=True, init=False,
             dtype="bf16"),
        # a training step of one layer
        dict(name="ssm_train", kind="ssm", train=True, B=4, S=2048, D=2048, N=16, G=1, gate=True, init=False, dtype="bf16"),
        # a small one in single precision, odd sizes, two groups of b and c, no gate, the state before given
        dict(name="ssm_train_f32", kind="ssm", train=True, B=2, S=501, D=300, N=24, G=2, gate=False, init=True, dtype="f32"),
    ]


def _log_int(rng, lo, hi):
    """An integer of [lo, hi], even over the logarithm."""
    lo, hi = max(1, lo), max(1, lo, hi)
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["norm", "norm", "conv", "conv", "conv_step", "ssm", "ssm", "ssm", "ssm_step"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "f32"])
    odd = rng.random() < 0.3   # widths that are no multiples of 8, else multiples of 64
    B = _log_int(rng, 1, 16)

    def width(lo, hi):
        w = _log_int(rng, lo, hi)
        return w | 1 if odd else max(64, w // 64 * 64)

    if kind == "norm":
        train, heads = rng.random() < 0.6, rng.random() < 0.5
        NH = rng.choice([4, 8, 16]) if heads else 1
        D = width(32, 512) if heads else width(32, 8192)
        S = _log_int(rng, 1, min(16384, (1 << 26) // (B * NH * D)))
        return dict(kind=kind, train=train, B=B, S=S, NH=NH, D=D, heads=heads, dtype=dtype, param=rng.choice([dtype, "f32"]))
    if kind == "conv_step":
        return dict(kind=kind, B=_log_int(rng, 1, 256), D=width(64, 8192), W=rng.choice([2, 3, 4, 4]), act=rng.random() < 0.7,
                    dtype=dtype)
    if kind == "conv":
        D = width(64, 4096)
        S = _log_int(rng, 1, min(16384, (1 << 25) // (B * D)))
        return dict(kind=kind, train=rng.random() < 0.6, B=B, S=S, D=D, W=rng.choice([2, 3, 4, 4]), act=rng.random() < 0.7,
                    init=rng.random() < 0.5, dtype=dtype)
    N = rng.choice([4, 8, 16, 16, 16, 32, 64, rng.randint(1, 64)])
    G = rng.choice([1, 1, 1, 2, 4])
    if kind == "ssm_step":
        B = _log_int(rng, 1, 256)
        D = width(64, max(64, min(8192, (1 << 23) // (B * N))))
        return dict(kind=kind, B=B, D=D * G if odd else D, N=N, G=G, dtype=dtype)
    train = rng.random() < 0.6
    D = width(64, 2048)
    D = D * G if odd else D
    S = _log_int(rng, 1, min(2048, (1 << 28) // (B * D * N)) if train else min(16384, (1 << 28) // (B * D * N)))
    return dict(kind=kind, train=train, B=B, S=S, D=D, N=N, G=G, gate=rng.random() < 0.7, init=rng.random() < 0.4, dtype=dtype)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dt = _DTYPE[case["dtype"]]
    f32 = torch.float32

    def randn(*shape, dtype=dt):
        return torch.randn(shape, generator=gen, device="cuda", dtype=f32).to(dtype)

    def rand(*shape):
        return torch.rand(shape, generator=gen, device="cuda", dtype=f32)

    s = dict(case=case)
    kind = case["kind"]
    if kind == "norm":
        B, S, NH, D = case["B"], case["S"], case["NH"], case["D"]
        pdt = _DTYPE[case["param"]]
        # values of a residual stream: other than zero in the mean, another scale for each token
        shape, row = ((B, NH, S, D), (B, NH, S, 1)) if case["heads"] else ((B, S, D), (B, S, 1))
        s["x"] = ((randn(*shape, dtype=f32) + 0.5 * randn(*row, dtype=f32)) * (0.25 + 2 * rand(*row))).to(dt)
        par = (NH, D) if case["heads"] else (D,)
        s["weight"] = (1 + 0.1 * randn(*par, dtype=f32)).to(pdt)
        s["bias"] = (0.1 * randn(*par, dtype=f32)).to(pdt)
        if case["train"]:
            s["dy"] = randn(B, S, NH, D) if case["heads"] else randn(B, S, D)
            s["leaves"] = [s[n].requires_grad_(True) for n in ("x", "weight", "bias")]
        return s
    B, D = case["B"], case["D"]
    if kind in ("conv", "conv_step"):
        W = case["W"]
        tok = (case["S"],) if kind == "conv" else ()
        s["x"] = randn(B, *tok, D)
        s["weight"] = ((2 * rand(D, W) - 1) * W ** -0.5).to(dt)
        s["bias"] = ((2 * rand(D) - 1) * W ** -0.5).to(dt)
        if kind == "conv_step" or case["init"]:
            s["before"] = randn(B, W - 1, D)
        if case.get("train"):
            s["dy"] = randn(B, *tok, D)
            s["leaves"] = [s[n].requires_grad_(True) for n in ("x", "weight", "bias", "before") if n in s]
        return s
    N, G = case["N"], case["G"]
    tok = (case["S"],) if kind == "ssm" else ()
    s["x"] = randn(B, *tok, D)
    s["dt"] = randn(B, *tok, D)
    if kind == "ssm_step" or case["gate"]:
        s["z"] = randn(B, *tok, D)
    s["b"] = randn(B, *tok, G, N)
    s["c"] = randn(B, *tok, G, N)
    # decay rates 1 ... N and time steps of 0.001 to 0.1, as such layers start out
    s["a"] = -(1.0 + torch.arange(N, device="cuda", dtype=f32)) * (0.8 + 0.4 * rand(D, N))
    step = torch.exp(math.log(1e-3) + rand(D) * (math.log(1e-1) - math.log(1e-3)))
    s["dt_bias"] = step + torch.log(-torch.expm1(-step))
    s["skip"] = 1 + 0.1 * randn(D, dtype=f32)
    if kind == "ssm_step" or case["init"]:
        s["h"] = randn(B, D, N, dtype=f32)
    if case.get("train"):
        s["dy"] = randn(B, *tok, D)
        s["leaves"] = [s[n].requires_grad_(True) for n in ("x", "dt", "a", "b", "c", "skip", "z", "dt_bias", "h") if n in s]
    return s


# ---- the plain forms ------------------------------------------------------------------------------------------------
def _silu(v):
    return v / (1 + torch.exp(-v))


def _softplus(v):
    return torch.where(v > 20, v, torch.log(1 + torch.exp(torch.clamp(v, max=20))))


def _plain_norm(x, weight, bias):
    v = x.float()
    v = v - v.mean(-1, keepdim=True)
    v = v / torch.sqrt((v * v).mean(-1, keepdim=True) + _EPS)
    return (v * weight.float() + bias.float()).to(x.dtype)


def _plain_conv(x, weight, bias, before, act):
    (B, S, D), W = x.shape, weight.shape[1]
    head = torch.zeros(B, W - 1, D, device=x.device) if before is None else before.float()
    v = torch.cat([head, x.float()], 1)
    w = weight.float()
    y = bias.float()
    for j in range(W):
        y = y + v[:, j:j + S] * w[:, j]
    y = _silu(y) if act else y
    return y.to(x.dtype), v[:, S:].to(x.dtype)


def _plain_ssm(s, backward):
    """Forward, and with `backward` the gradients of all leaves, with every state kept."""
    x, a, b, c = s["x"].detach().float(), s["a"].detach(), s["b"].detach().float(), s["c"].detach().float()
    (B, S, D), (G, N) = x.shape, b.shape[2:]
    heads = lambda v: v.view(*v.shape[:-1], G, D // G)  # noqa: E731
    raw = s["dt"].detach().float() + s["dt_bias"].detach()
    step = _softplus(raw)
    a_g = a.view(G, D // G, N)
    tx = (lambda v: v.transpose(0, 1))  # time first
    decay = torch.exp(heads(tx(step))[..., None] * a_g)
    inc = heads(tx(step * x))[..., None] * tx(b)[:, :, :, None, :]
    h = s["h"].detach().view(B, G, D // G, N) if "h" in s else torch.zeros(B, G, D // G, N, device=x.device)
    states = torch.empty(S + 1, B, G, D // G, N, device=x.device)
    states[0] = h
    for t in range(S):
        h = decay[t] * h + inc[t]
        states[t + 1] = h
    del inc
    cs = tx(c)[:, :, :, None, :]
    skip = s["skip"].detach()
    out = tx((states[1:] * cs).sum(-1).reshape(S, B, D)) + skip * x
    z = s["z"].detach().float() if "z" in s else None
    y = out if z is None else out * _silu(z)
    r = {"y": y.to(s["x"].dtype), "h": h.reshape(B, D, N)}
    if not backward:
        return r
    dy = s["dy"].float()
    dout = dy if z is None else dy * _silu(z)
    dout_t = heads(tx(dout))[..., None]
    g = torch.zeros(B, G, D // G, N, device=x.device)
    grads = torch.empty(S, B, G, D // G, N, device=x.device)
    for t in range(S - 1, -1, -1):
        g = dout_t[t] * cs[t] + g
        grads[t] = g
        g = decay[t] * g
    grad = {"h": g.reshape(B, D, N)}
    grad["c"] = tx((states[1:] * dout_t).sum(3))
    grad["b"] = tx((grads * heads(tx(step * x))[..., None]).sum(3))
    through = grads * decay * states[:-1]
    grad["a"] = (through * heads(tx(step))[..., None]).sum((0, 1)).view(D, N)
    flat = lambda v: tx(v.reshape(S, B, D))  # noqa: E731
    gb = flat((grads * tx(b)[:, :, :, None, :]).sum(-1))
    draw_ = (flat((through * a_g).sum(-1)) + x * gb) / (1 + torch.exp(-raw))
    grad["x"] = step * gb + skip * dout
    grad["dt"], grad["dt_bias"] = draw_, draw_.sum((0, 1))
    grad["skip"] = (dout * x).sum((0, 1))
    if z is not None:
        sig = 1 / (1 + torch.exp(-z))
        grad["z"] = dy * out * sig * (1 + z * (1 - sig))
    for n in ("x", "dt", "a", "b", "c", "skip", "z", "dt_bias", "h"):
        if n in s:
            r["d" + n] = grad[n].to(s[n].dtype)
    return r


def _run_plain(s):
    case = s["case"]
    kind = case["kind"]
    if kind == "norm":
        x = s["x"].transpose(1, 2) if case["heads"] else s["x"]
        if not case["train"]:
            return {"y": _plain_norm(x, s["weight"], s["bias"])}
        y = _plain_norm(x, s["weight"], s["bias"])
        return {"y": y, **dict(zip(("dx", "dweight", "dbias"), torch.autograd.grad(y, s["leaves"], s["dy"])))}
    if kind == "conv_step":
        y, last = _plain_conv(s["x"][:, None], s["weight"], s["bias"], s["before"], case["act"])
        return {"y": y[:, 0], "before": last}
    if kind == "conv":
        y, last = _plain_conv(s["x"], s["weight"], s["bias"], s.get("before"), case["act"])
        if not case["train"]:
            return {"y": y, "last": last}
        return {"y": y, **dict(zip(("dx", "dweight", "dbias", "dbefore"), torch.autograd.grad(y, s["leaves"], s["dy"])))}
    if kind == "ssm_step":
        x = s["x"].float()
        (B, D), (G, N) = x.shape, s["b"].shape[1:]
        step = _softplus(s["dt"].float() + s["dt_bias"])
        wide = lambda v: v.float().repeat_interleave(D // G, 1)  # noqa: E731
        h = torch.exp(step[..., None] * s["a"]) * s["h"] + (step * x)[..., None] * wide(s["b"])
        y = ((h * wide(s["c"])).sum(-1) + s["skip"] * x) * _silu(s["z"].float())
        return {"y": y.to(s["x"].dtype), "h": h}
    return _plain_ssm(s, case["train"])


# ---- the framework's operators --------------------------------------------------------------------------------------
def _run_own(s):
    import mlstm_kernels_b200 as mk
    case = s["case"]
    kind = case["kind"]
    if kind == "norm":
        x = s["x"].transpose(1, 2) if case["heads"] else s["x"]
        y = mk.layer_norm__b200(x, s["weight"], s["bias"], eps=_EPS)
        if not case["train"]:
            return {"y": y}
        return {"y": y, **dict(zip(("dx", "dweight", "dbias"), torch.autograd.grad(y, s["leaves"], s["dy"])))}
    act = "silu" if case.get("act") else None
    if kind == "conv_step":
        y, before = mk.short_conv_step__b200(s["x"], s["before"], s["weight"], s["bias"], activation=act)
        return {"y": y, "before": before}
    if kind == "conv":
        if not case["train"]:
            y, last = mk.short_conv__b200(s["x"], s["weight"], s["bias"], s.get("before"), return_last_states=True,
                                          activation=act)
            return {"y": y, "last": last}
        y = mk.short_conv__b200(s["x"], s["weight"], s["bias"], s.get("before"), activation=act)
        return {"y": y, **dict(zip(("dx", "dweight", "dbias", "dbefore"), torch.autograd.grad(y, s["leaves"], s["dy"])))}
    if kind == "ssm_step":
        y, h = mk.ssm_step__b200(s["x"], s["dt"], s["a"], s["b"], s["c"], s["h"], skip=s["skip"], z=s["z"],
                                 dt_bias=s["dt_bias"], softplus=True)
        return {"y": y, "h": h}
    y, h = mk.ssm_scan__b200(s["x"], s["dt"], s["a"], s["b"], s["c"], skip=s["skip"], z=s.get("z"), dt_bias=s["dt_bias"],
                             softplus=True, h_initial=s.get("h"), return_last_states=True)
    r = {"y": y, "h": h.detach()}
    if case["train"]:
        names = [n for n in ("x", "dt", "a", "b", "c", "skip", "z", "dt_bias", "h") if n in s]
        r.update(zip(("d" + n for n in names), torch.autograd.grad(y, s["leaves"], s["dy"])))
    return r


def run(s):
    return _run_own(s) if own else _run_plain(s)


# ---- the definitions in 64 bits -------------------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    q = {n: v.detach().double() for n, v in s.items() if isinstance(v, torch.Tensor)}
    kind = case["kind"]
    x = q["x"]
    if kind == "norm":
        if case["heads"]:
            x = x.permute(0, 2, 1, 3)
        var, mu = torch.var_mean(x, -1, correction=0, keepdim=True)
        r = (var + _EPS).rsqrt()
        n = (x - mu) * r
        out = {"y": n * q["weight"] + q["bias"]}
        if case["train"]:
            dn = q["dy"] * q["weight"]
            dx = r * (dn - dn.mean(-1, keepdim=True) - n * (dn * n).mean(-1, keepdim=True))
            out["dx"] = dx.permute(0, 2, 1, 3) if case["heads"] else dx
            out["dweight"], out["dbias"] = (q["dy"] * n).sum((0, 1)), q["dy"].sum((0, 1))
        return out
    if kind in ("conv", "conv_step"):
        step = kind == "conv_step"
        x = x[:, None] if step else x
        (B, S, D), W = x.shape, case["W"]
        v = x.new_zeros(B, W - 1 + S, D)
        v[:, W - 1:] = x
        if "before" in q:
            v[:, :W - 1] = q["before"]
        u = (v.unfold(1, W, 1) * q["weight"]).sum(-1) + q["bias"]   # windows (B, S, D, W)
        y = u * torch.sigmoid(u) if case["act"] else u
        if step:
            return {"y": y[:, 0], "before": v[:, 1:]}
        if not case["train"]:
            return {"y": y, "last": v[:, S:]}
        p = torch.sigmoid(u)
        du = q["dy"] * p * (1 + u * (1 - p)) if case["act"] else q["dy"]
        dv = torch.zeros_like(v)
        for j in range(W):
            dv[:, j:j + S] += du * q["weight"][:, j]
        out = {"y": y, "dx": dv[:, W - 1:], "dbias": du.sum((0, 1)),
               "dweight": torch.stack([(du * v[:, j:j + S]).sum((0, 1)) for j in range(W)], -1)}
        if "before" in q:
            out["dbefore"] = dv[:, :W - 1]
        return out
    D, N, G = case["D"], case["N"], case["G"]
    B = x.shape[0]
    group = torch.arange(D, device=x.device) // (D // G)   # of each channel
    if kind == "ssm_step":
        q = {n: v[:, None] if n in ("x", "dt", "z", "b", "c") else v for n, v in q.items()}
        x = q["x"]
    S = x.shape[1]
    raw = q["dt"] + q["dt_bias"]
    step = torch.logaddexp(raw, torch.zeros_like(raw))
    h = q["h"].clone() if "h" in q else x.new_zeros(B, D, N)
    out = x.new_empty(B, S, D)
    kept = [h]
    for t in range(S):
        h = torch.exp(step[:, t, :, None] * q["a"]) * h + (step[:, t] * x[:, t])[..., None] * q["b"][:, t, group]
        out[:, t] = torch.einsum("bdn,bdn->bd", h, q["c"][:, t, group]) + q["skip"] * x[:, t]
        if case.get("train"):
            kept.append(h)
    y = out * q["z"] * torch.sigmoid(q["z"]) if "z" in q else out
    if kind == "ssm_step":
        return {"y": y[:, 0], "h": h}
    res = {"y": y, "h": h}
    if not case["train"]:
        return res
    if "z" in q:
        p = torch.sigmoid(q["z"])
        res["dz"] = q["dy"] * out * (p + q["z"] * p * (1 - p))
        dout = q["dy"] * q["z"] * p
    else:
        dout = q["dy"]
    d = {n: torch.zeros_like(v) for n, v in q.items()}
    g = torch.zeros_like(h)
    by_group = torch.zeros(D, G, device=x.device, dtype=x.dtype)
    by_group[torch.arange(D, device=x.device), group] = 1
    for t in range(S - 1, -1, -1):
        dec = torch.exp(step[:, t, :, None] * q["a"])
        g = g + dout[:, t, :, None] * q["c"][:, t, group]
        d["c"][:, t] = torch.einsum("bdn,dg->bgn", kept[t + 1] * dout[:, t, :, None], by_group)
        d["b"][:, t] = torch.einsum("bdn,dg->bgn", g * (step[:, t] * x[:, t])[..., None], by_group)
        gb = torch.einsum("bdn,bdn->bd", g, q["b"][:, t, group])
        back = g * dec
        rate = back * kept[t]
        d["x"][:, t] = step[:, t] * gb + q["skip"] * dout[:, t]
        d["dt"][:, t] = torch.einsum("bdn,dn->bd", rate, q["a"]) + x[:, t] * gb
        d["a"] += torch.einsum("bdn,bd->dn", rate, step[:, t])
        g = back
        kept.pop()
    d["dt"] = d["dt"] * torch.sigmoid(raw)
    d["dt_bias"] = d["dt"].sum((0, 1))
    d["skip"] = (dout * x).sum((0, 1))
    d["h"] = g
    for n in ("x", "dt", "a", "b", "c", "skip", "dt_bias", "h"):
        if n in s:
            res["d" + n] = d[n]
    return res


def work(case):
    el = _BYTES[case["dtype"]]
    kind, B = case["kind"], case["B"]
    S, train = case.get("S", 1), case.get("train", False)
    if kind == "norm":
        n, par = B * S * case["NH"] * case["D"], 2 * case["NH"] * case["D"] * _BYTES[case["param"]]
        # forward: mean, squares, scale and shift; backward: two means, two sums over the tokens
        return {"bytes": n * el * (4 if train else 2) + par * (2 if train else 1), "flops": n * (20 if train else 7)}
    D = case["D"]
    n = B * S * D
    if kind in ("conv", "conv_step"):
        W, par = case["W"], D * (case["W"] + 1) * el
        kept = B * (W - 1) * D * el
        flops = n * (2 * W + (4 if case["act"] else 0))
        if not train:
            return {"bytes": 2 * n * el + par + kept * (2 if "S" not in case or case["init"] else 1), "flops": flops}
        return {"bytes": 4 * n * el + 2 * par + (2 * kept if case["init"] else 0),
                "flops": 2 * flops + n * (4 * W + (8 if case["act"] else 0))}
    N, G = case["N"], case["G"]
    gate = 1 if kind == "ssm_step" or case["gate"] else 0
    init = kind == "ssm_step" or case["init"]
    tok, bc, par, state = n * el, 2 * B * S * G * N * el, D * (N + 2) * 4, B * D * N * 4
    # per state and token: exponent, exponential, increment, decay and add, output
    flops = n * (7 * N + 8)
    if not train:
        return {"bytes": (3 + gate) * tok + bc + par + state * (2 if init else 1), "flops": flops}
    # x, dt, z, dy in, y and three gradients out; per state and token of the backward: the adjoint, four products summed
    return {"bytes": (6 + 2 * gate) * tok + 2 * bc + 2 * par + state * (3 if init else 1), "flops": 2 * flops + n * (13 * N + 16)}
