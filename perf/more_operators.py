"""A gated linear recurrence with its step for single tokens, and dropout without a stored mask, as cases that can be timed and
compared.

Where `own` is false, run() computes them from elementary torch operations; where it is true, through this package.

  scan        h_t = a_t h_{t-1} + s(a_t) sigmoid(i_t) x_t per channel, y_t = h_t silu(z_t), over x, f, i, z (B, S, D);
              a = sigmoid(f), or exp(rate sigmoid(f)) with a rate (D,); s(a) = 1, 1 - a ("convex") or sqrt(1 - a^2) ("variance");
              step is one token of it
  dropout     y = residual + (w_n >= p 2^32 ? x / (1 - p) : 0), w_n the n-th 32-bit word of a counter-based generator
              (Philox4x32 with 7 rounds; Salmon, Moraes, Dror, Shaw: Parallel random numbers, 2011): word n mod 4 of the counter
              (n div 4, offset) under the key `seed`, n the index of the element in x
"""

import math

import torch

own = False

_DTYPE = {"bf16": torch.bfloat16, "fp16": torch.float16, "f32": torch.float32}
_BYTES = {"bf16": 2, "fp16": 2, "f32": 4}


def listed():
    return [
        # one token of four users: the smallest call, launch latency and host time count
        dict(name="step_few", kind="step", B=4, D=2048, i=True, z=False, rate=True, scale="variance", dtype="bf16"),
        # one token of a serving batch with every gate
        dict(name="step_many", kind="step", B=512, D=4096, i=True, z=True, rate=False, scale="convex", dtype="bf16"),
        # a prompt of any length: one gate for what is kept and what is added
        dict(name="scan_prompt_fp16", kind="scan", train=False, B=1, S=8077, D=2048, i=False, z=False, rate=False, scale="convex",
             init=False, dtype="fp16"),
        # one long document in a layer of few channels
        dict(name="scan_document", kind="scan", train=False, B=1, S=65536, D=2048, i=True, z=False, rate=True, scale="variance",
             init=False, dtype="bf16"),
        # a training step of one layer, 32 768 tokens
        dict(name="scan_train", kind="scan", train=True, B=8, S=4096, D=2048, i=True, z=False, rate=True, scale="variance",
             init=False, dtype="bf16"),
        # the same tokens in longer sequences and a wider layer, with an output gate: the largest
        dict(name="scan_train_gated", kind="scan", train=True, B=4, S=8192, D=4096, i=False, z=True, rate=False, scale="convex",
             init=False, dtype="bf16"),
        # segments of longer texts in single precision: odd sizes, separate gates, the state before given
        dict(name="scan_train_f32", kind="scan", train=True, B=3, S=777, D=1001, i=True, z=False, rate=False, scale=None,
             init=True, dtype="f32"),
        # a small model's residual branch: launch latency and host time count
        dict(name="dropout_small", kind="dropout", train=True, B=1, S=128, NH=1, D=512, heads=False, p=0.1,
             residual="same", dtype="bf16"),
        # the residual branch of a training step, 32 768 tokens
        dict(name="dropout_train", kind="dropout", train=True, B=8, S=4096, NH=1, D=2048, heads=False, p=0.1,
             residual="same", dtype="bf16"),
        # a wide layer whose residual stream is kept in single precision
        dict(name="dropout_train_stream", kind="dropout", train=True, B=4, S=8192, NH=1, D=4096, heads=False, p=0.2,
             residual="f32", dtype="bf16"),
        # the heads of a recurrence, (B, NH, S, DH) read as (B, S, NH, DH), in a pass whose gradients come later
        dict(name="dropout_heads_fp16", kind="dropout", train=False, B=4, S=4096, NH=16, D=256, heads=True, p=0.1,
             residual=None, dtype="fp16"),
        # odd sizes in single precision
        dict(name="dropout_train_f32", kind="dropout", train=True, B=3, S=777, NH=1, D=1001, heads=False, p=0.5,
             residual="same", dtype="f32"),
    ]


def _log_int(rng, lo, hi):
    """An integer of [lo, hi], even over the logarithm."""
    lo, hi = max(1, lo), max(1, lo, hi)
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["scan", "scan", "scan", "scan", "step", "dropout", "dropout"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "f32"])
    odd = rng.random() < 0.3   # widths that are no multiples of 8, else multiples of 64
    B = _log_int(rng, 1, 16)

    def width(lo, hi):
        w = _log_int(rng, lo, hi)
        return w | 1 if odd else max(64, w // 64 * 64)

    if kind == "dropout":
        heads = rng.random() < 0.3
        NH = rng.choice([4, 8, 16]) if heads else 1
        D = width(32, 512) if heads else width(64, 8192)
        S = _log_int(rng, 1, min(16384, (1 << 25) // (B * NH * D)))
        return dict(kind=kind, train=rng.random() < 0.6, B=B, S=S, NH=NH, D=D, heads=heads,
                    p=rng.choice([0.05, 0.1, 0.1, 0.2, 0.5]), residual=rng.choice([None, "same", "same", "f32"]), dtype=dtype)
    gates = dict(i=rng.random() < 0.6, z=rng.random() < 0.4, rate=rng.random() < 0.5, scale=rng.choice([None, "convex", "variance"]))
    if kind == "step":
        return dict(kind=kind, B=_log_int(rng, 1, 512), D=width(64, 8192), dtype=dtype, **gates)
    D = width(64, 4096)
    S = _log_int(rng, 1, min(65536, (1 << 25) // (B * D)))
    return dict(kind=kind, train=rng.random() < 0.6, B=B, S=S, D=D, init=rng.random() < 0.4, dtype=dtype, **gates)


_LEAVES = ("x", "f", "i", "z", "rate", "h")


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dt = _DTYPE[case["dtype"]]
    f32 = torch.float32

    def randn(*shape, dtype=dt):
        return torch.randn(shape, generator=gen, device="cuda", dtype=f32).to(dtype)

    def rand(*shape):
        return torch.rand(shape, generator=gen, device="cuda", dtype=f32)

    s = dict(case=case)
    if case["kind"] == "dropout":
        B, S, NH, D = case["B"], case["S"], case["NH"], case["D"]
        shape, seen = ((B, NH, S, D), (B, S, NH, D)) if case["heads"] else ((B, S, D), (B, S, D))
        s["x"] = randn(*shape)
        rdt = f32 if case["residual"] == "f32" else dt
        if case["residual"]:
            s["residual"] = randn(*seen, dtype=rdt)
        # the generator's key lies on the GPU, as a captured training step has it; the layer's number is known to the host
        s["seed"] = torch.tensor([(seed * 0x9E3779B97F4A7C15 + 1) % (1 << 63)], device="cuda")
        s["offset"] = 3 + seed % 5
        if case["train"]:
            s["dy"] = randn(*seen, dtype=rdt)
            s["leaves"] = [s[n].requires_grad_(True) for n in ("x", "residual") if n in s]
        return s
    B, D = case["B"], case["D"]
    tok = (case["S"],) if case["kind"] == "scan" else ()
    s["x"] = randn(B, *tok, D)
    if case["rate"]:
        # decays of 0.6 to 0.99 where the gate is open, up to 0.999 where it is nearly closed
        s["f"] = randn(B, *tok, D)
        s["rate"] = -torch.exp(math.log(1e-2) + rand(D) * (math.log(0.5) - math.log(1e-2)))
    else:
        # each channel with a span of its own, from a token to some hundreds
        s["f"] = (randn(B, *tok, D, dtype=f32) + 6 * rand(D)).to(dt)
    if case["i"]:
        s["i"] = randn(B, *tok, D)
    if case["z"]:
        s["z"] = randn(B, *tok, D)
    if case["kind"] == "step" or case["init"]:
        s["h"] = randn(B, D, dtype=f32)
    if case.get("train"):
        s["dy"] = randn(B, *tok, D)
        s["leaves"] = [s[n].requires_grad_(True) for n in _LEAVES if n in s]
    return s


# ---- the plain forms ------------------------------------------------------------------------------------------------
def _sigmoid(v):
    return 1 / (1 + torch.exp(-v))


def _decay(s):
    """sigmoid(f), log a, a, 1 - a, 1 - a^2"""
    f = s["f"].detach().float()
    sf = _sigmoid(f)
    if "rate" in s:
        r = s["rate"].detach() * sf
        return sf, r, torch.exp(r), -torch.expm1(r), -torch.expm1(2 * r)
    rest = _sigmoid(-f)
    return sf, None, sf, rest, rest * (1 + sf)


def _scan(a, u):
    """h_t = a_t h_{t-1} + u_t along axis 1, by doubling the tokens that are joined; overwrites both."""
    S, d = u.shape[1], 1
    while d < S:
        u[:, d:] += a[:, d:] * u[:, :-d]
        a[:, d:] = a[:, d:] * a[:, :-d]
        d *= 2
    return u


def _input_scale(s, a, rest, rest2):
    scale = s["case"]["scale"]
    return torch.ones_like(a) if scale is None else rest if scale == "convex" else torch.sqrt(rest2)


def _plain_scan(s, backward):
    x = s["x"].detach().float()
    x, seq = (x, True) if x.dim() == 3 else (x[:, None], False)
    sf, r, a, rest, rest2 = (v if v is None or seq else v[:, None] for v in _decay(s))
    sx = _input_scale(s, a, rest, rest2)
    si = _sigmoid(s["i"].detach().float().view_as(x)) if "i" in s else None
    g = sx if si is None else sx * si
    u = g * x
    h0 = s["h"].detach() if "h" in s else torch.zeros_like(x[:, 0])
    h = u.clone()
    h[:, 0] += a[:, 0] * h0
    h = _scan(a.clone(), h)
    z = s["z"].detach().float().view_as(x) if "z" in s else None
    sz = None if z is None else _sigmoid(z)
    y = h if z is None else h * (z * sz)
    res = {"y": (y if seq else y[:, 0]).to(s["x"].dtype), "h": h[:, -1].clone()}
    if not backward:
        return res
    dy = s["dy"].float()
    G = dy.clone() if z is None else dy * (z * sz)
    back = torch.zeros_like(a)
    back[:, 1:] = a[:, 1:].flip(1)      # of the reversed tokens: a_{t+1}
    G = _scan(back, G.flip(1)).flip(1)
    hp = torch.cat([h0[:, None], h[:, :-1]], 1)
    scale = s["case"]["scale"]
    d = {"x": G * g, "h": a[:, 0] * G[:, 0]}
    if si is not None:
        d["i"] = G * u * (1 - si)
    if z is not None:
        d["z"] = dy * h * (sz * (1 + z * (1 - sz)))
    if r is None:
        l = 0 if scale is None else -a if scale == "convex" else -a * a / (1 + a)
        d["f"] = G * (a * rest * hp + u * l)
    else:
        k = 0 if scale is None else -r * a / rest if scale == "convex" else -r * a * a / rest2
        d["f"] = G * _sigmoid(-s["f"].detach().float()) * (r * a * hp + u * k)
        d["rate"] = (G * (sf * a * hp + u * k / s["rate"].detach())).sum((0, 1))
    for n in _LEAVES:
        if n in s:
            res["d" + n] = d[n].to(s[n].dtype)
    return res


_LOW = 0xFFFFFFFF


def _words(count, seed, offset):
    """The first `count` words; the products of two 32-bit numbers wrap around in 64 bits, which leaves all of theirs."""
    n = torch.arange((count + 3) // 4, device=seed.device)
    c = [n & _LOW, n >> 32, torch.full_like(n, offset & _LOW), torch.full_like(n, offset >> 32)]
    k0, k1 = seed & _LOW, (seed >> 32) & _LOW
    for _ in range(7):
        p0, p1 = c[0] * 0xD2511F53, c[2] * 0xCD9E8D57
        c = [((p1 >> 32) & _LOW) ^ c[1] ^ k0, p1 & _LOW, ((p0 >> 32) & _LOW) ^ c[3] ^ k1, p0 & _LOW]
        k0, k1 = (k0 + 0x9E3779B9) & _LOW, (k1 + 0xBB67AE85) & _LOW
    return torch.stack(c, -1).flatten()[:count]


def _plain_dropout(s):
    case = s["case"]
    x = s["x"].detach().transpose(1, 2) if case["heads"] else s["x"].detach()
    p = case["p"]
    keep = (_words(x.numel(), s["seed"], s["offset"]) >= round(p * 2.0 ** 32)).view(x.shape)
    y = torch.where(keep, x.float() * (1 / (1 - p)), 0.0)
    if "residual" in s:
        y = y + s["residual"].detach().float()
    res = {"y": y.to(torch.float32 if case["residual"] == "f32" else x.dtype)}
    if case["train"]:
        dx = torch.where(keep, s["dy"].float() * (1 / (1 - p)), 0.0).to(x.dtype)
        res["dx"] = dx.transpose(1, 2) if case["heads"] else dx
        if "residual" in s:
            res["dresidual"] = s["dy"].clone()
    return res


def _run_plain(s):
    if s["case"]["kind"] == "dropout":
        return _plain_dropout(s)
    return _plain_scan(s, s["case"].get("train", False))


# ---- the framework's operators --------------------------------------------------------------------------------------
def _run_own(s):
    import mlstm_kernels_b200 as mk
    case = s["case"]
    if case["kind"] == "dropout":
        x = s["x"].transpose(1, 2) if case["heads"] else s["x"]
        y = mk.dropout__b200(x, case["p"], s["seed"], offset=s["offset"], residual=s.get("residual"))
        if not case["train"]:
            return {"y": y}
        names = [n for n in ("dx", "dresidual") if n[1:] in s]
        return {"y": y, **dict(zip(names, torch.autograd.grad(y, s["leaves"], s["dy"])))}
    gates = dict(i=s.get("i"), z=s.get("z"), rate=s.get("rate"), input_scale=case["scale"])
    if case["kind"] == "step":
        y, h = mk.gated_step__b200(s["x"], s["f"], s["h"], **gates)
        return {"y": y, "h": h}
    y, h = mk.gated_scan__b200(s["x"], s["f"], h_initial=s.get("h"), return_last_states=True, **gates)
    r = {"y": y, "h": h.detach()}
    if case["train"]:
        r.update(zip(("d" + n for n in _LEAVES if n in s), torch.autograd.grad(y, s["leaves"], s["dy"])))
    return r


def run(s):
    return _run_own(s) if own else _run_plain(s)


# ---- the definitions in 64 bits -------------------------------------------------------------------------------------
def _halves(a, b):
    """a b of 32-bit numbers as (high, low) 32 bits, from products of 16-bit numbers."""
    al, ah, bl, bh = a % 65536, a // 65536, b % 65536, b // 65536
    mid = ah * bl + (al * bl) // 65536
    mid2 = al * bh + mid % 65536
    return ah * bh + mid // 65536 + mid2 // 65536, (mid2 % 65536) * 65536 + (al * bl) % 65536


def _exact_keep(count, seed, offset, p):
    m0, m1, mod = 0xD2511F53, 0xCD9E8D57, 1 << 32
    out = torch.empty((count + 3) // 4 * 4, dtype=torch.bool, device="cuda")
    step = 1 << 22
    for start in range(0, (count + 3) // 4, step):
        n = torch.arange(start, min(start + step, (count + 3) // 4), device="cuda")
        x0, x1 = n % mod, n // mod
        x2, x3 = torch.full_like(n, offset % mod), torch.full_like(n, offset // mod)
        for i in range(7):
            k0, k1 = (seed % mod + i * 0x9E3779B9) % mod, (seed // mod + i * 0xBB67AE85) % mod
            h0, l0 = _halves(x0, m0)
            h1, l1 = _halves(x2, m1)
            x0, x1, x2, x3 = h1 ^ x1 ^ k0, l1, h0 ^ x3 ^ k1, l0
        out[4 * start:4 * start + 4 * n.numel()] = (torch.stack([x0, x1, x2, x3], 1) >= round(p * mod)).flatten()
    return out[:count]


def exact(case, seed):
    s = prepare(case, seed)
    q = {n: v.detach().double() for n, v in s.items() if isinstance(v, torch.Tensor) and n != "seed"}
    if case["kind"] == "dropout":
        x = q["x"].permute(0, 2, 1, 3) if case["heads"] else q["x"]
        keep = _exact_keep(x.numel(), int(s["seed"]), s["offset"], case["p"]).view(x.shape)
        out = {"y": keep * x / (1 - case["p"]) + q.get("residual", 0)}
        if case["train"]:
            dx = keep * q["dy"] / (1 - case["p"])
            out["dx"] = dx.permute(0, 2, 1, 3) if case["heads"] else dx
            if "residual" in q:
                out["dresidual"] = q["dy"]
        return out
    step = case["kind"] == "step"
    t_first = lambda v: v[None] if step else v.transpose(0, 1)  # noqa: E731
    x, f, i, z, dy = (t_first(q[n]) if n in q else None for n in ("x", "f", "i", "z", "dy"))
    S, scale = x.shape[0], case["scale"]
    h = q["h"] if "h" in q else torch.zeros_like(x[0])
    first = h
    gate = torch.ones_like(x) if i is None else torch.sigmoid(i)
    sf = torch.sigmoid(f)
    log_a = q["rate"] * sf if case["rate"] else torch.nn.functional.logsigmoid(f)
    a = torch.exp(log_a)
    rest = -torch.expm1(log_a)                       # 1 - a
    sc = torch.ones_like(a) if scale is None else rest if scale == "convex" else torch.sqrt(rest * (1 + a))
    hs = torch.empty_like(x)
    u = sc * gate * x
    for t in range(S):
        h = a[t] * h + u[t]
        hs[t] = h
    o = torch.ones_like(x) if z is None else z * torch.sigmoid(z)
    back = (lambda v: v[0]) if step else (lambda v: v.transpose(0, 1))
    out = {"y": back(hs * o), "h": h}
    if not case.get("train"):
        return out
    G = torch.empty_like(x)
    g = torch.zeros_like(h)
    direct = dy * o
    for t in range(S - 1, -1, -1):
        G[t] = direct[t] + g
        g = a[t] * G[t]
    before = torch.cat([first[None], hs[:-1]])
    d = {"x": G * sc * gate, "h": g}
    if i is not None:
        d["i"] = G * sc * x * gate * (1 - gate)
    if z is not None:
        sz = torch.sigmoid(z)
        d["z"] = dy * hs * (sz + z * sz * (1 - sz))
    # through a: h_{t-1}, and the derivative of the scale
    d_scale = 0 if scale is None else -1 if scale == "convex" else -a / sc
    d_log = G * (before + d_scale * gate * x) * a
    if case["rate"]:
        d["f"] = d_log * q["rate"] * sf * (1 - sf)
        d["rate"] = (d_log * sf).sum((0, 1))
    else:
        d["f"] = d_log * torch.sigmoid(-f)
    for n in _LEAVES:
        if n in s:
            out["d" + n] = back(d[n]) if n in ("x", "f", "i", "z") else d[n]
    return out


def work(case):
    el = _BYTES[case["dtype"]]
    if case["kind"] == "dropout":
        n = case["B"] * case["S"] * case["NH"] * case["D"]
        rel = {None: 0, "same": el, "f32": 4}[case["residual"]]
        y = rel or el
        # a counter's seven rounds for four elements, comparison and scale; the gradient of the residual is that of y itself
        return {"bytes": n * (el + rel + y) + (n * (y + el) if case["train"] else 0), "flops": n * (13 if case["train"] else 12)}
    B, D, S, train = case["B"], case["D"], case.get("S", 1), case.get("train", False)
    n = B * S * D
    ins = 2 + case["i"] + case["z"]
    init = case["kind"] == "step" or case["init"]
    state, par = B * D * 4, D * 4 * case["rate"]
    flops = n * (6 + 4 * case["i"] + 5 * case["z"] + 3 * case["rate"] + (3 if case["scale"] else 0))
    if not train:
        return {"bytes": n * el * (ins + 1) + par + state * (1 + init), "flops": flops}
    # the inputs, y, dy and the inputs' gradients
    return {"bytes": n * el * (2 * ins + 2) + 2 * par + state * (1 + 2 * init), "flops": 3 * flops}
