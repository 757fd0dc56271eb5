"""Timing cases of the sequence-block operators: layer norm, linear with a fused epilogue, gated linear recurrence.

`prepare` makes a case's inputs, `run` makes one pass through the operator: with `own` set through vae_amd.layers, else in plain
form (elementary torch operations in 32 bits, one rounding at the end).  `exact` gives the same outputs in 64 bits.
"""
import math

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
ESIZE = {"f32": 4, "bf16": 2, "f16": 2}


# ----------------------------------------------------------------------------------------------- cases
def _norm(name, rows, cols, dtype, wdtype, train):
    return dict(name=name, op="norm", rows=rows, cols=cols, dtype=dtype, wdtype=wdtype, train=train)


def _linear(name, m, n, k, dtype, act, bias, residual, train):
    return dict(name=name, op="linear", m=m, n=n, k=k, dtype=dtype, act=act, bias=bias, residual=residual, train=train)


def _scan(name, b, t, d, dtype, ragged, train):
    return dict(name=name, op="scan", b=b, t=t, d=d, dtype=dtype, ragged=ragged, train=train)


def listed():
    return [
        # one token of a served model: the call's own latency
        _norm("norm_token_bf16", 1, 4096, "bf16", "bf16", False),
        # every step of a batch of 4096 windows of 60 steps at the series models' hidden size of 30 (rows of 120 bytes)
        _norm("norm_windows_f32", 4096 * 60, 30, "f32", "f32", True),
        # a training step over 65,536 positions, parameters kept in fp32
        _norm("norm_train_bf16", 65536, 1024, "bf16", "f32", True),
        # wide rows whose length is odd (no row but the first is aligned)
        _norm("norm_odd_f16", 2047, 8195, "f16", "f16", True),
        # one token through a square layer: the weights' bytes are the bound
        _linear("linear_token_bf16", 1, 4096, 4096, "bf16", "silu", True, True, False),
        # the 288 -> 100 hidden layer of the image model's heads at its training batch
        _linear("linear_heads_f32", 4096, 100, 288, "f32", "leaky", True, False, True),
        # a training step of a block's layer over 16,384 positions
        _linear("linear_train_bf16", 16384, 4096, 4096, "bf16", "gelu", True, True, True),
        # a ragged batch through a layer of odd sizes
        _linear("linear_odd_f16", 1537, 1001, 1283, "f16", "leaky", True, True, True),
        # one step of 256 streams: the state in, the state out
        _scan("scan_token_bf16", 256, 1, 2048, "bf16", False, False),
        # a batch of 4096 windows of up to 60 steps at hidden size 30
        _scan("scan_windows_f32", 4096, 60, 30, "f32", True, True),
        # an ordinary training step
        _scan("scan_train_bf16", 8, 4096, 2048, "bf16", False, True),
        # one long series: few channels, the time axis carries the parallelism
        _scan("scan_long_f32", 1, 65521, 512, "f32", False, True),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    op = rng.choice(["norm", "linear", "scan"])
    dtype = rng.choice(["f32", "bf16", "f16"])
    train = rng.random() < 0.7
    if op == "norm":
        cols = _log_int(rng, 8, 16384)
        rows = _log_int(rng, 1, min(262144, 2 ** 26 // cols))
        case = _norm("", rows, cols, dtype, rng.choice(["f32", dtype]), train)
    elif op == "linear":
        n, k = _log_int(rng, 8, 8192), _log_int(rng, 8, 8192)
        if rng.random() < 0.5:  # half of the layers have sizes that are multiples of 16, as a user chooses them
            n, k = -(-n // 16) * 16, -(-k // 16) * 16
        m = _log_int(rng, 1, min(16384, 2 ** 38 // (n * k)))
        case = _linear("", m, n, k, dtype, rng.choice(["none", "leaky", "sigmoid", "gelu", "silu"]), rng.random() < 0.7,
                       rng.random() < 0.5, train)
    else:
        d = _log_int(rng, 8, 4096)
        b = _log_int(rng, 1, min(4096, 2 ** 26 // d))
        t = _log_int(rng, 1, min(65536, 2 ** 26 // (b * d)))
        case = _scan("", b, t, d, dtype, rng.random() < 0.5, train)
    del case["name"]
    return case


# ---------------------------------------------------------------------------------------------- inputs
EPS = 1e-5
SLOPE = 0.2  # of "leaky": the series models' slope


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = DTYPES[case["dtype"]]

    def randn(*shape, scale=1.0, mean=0.0, dtype=dt):
        return (torch.randn(*shape, generator=g, device="cuda") * scale + mean).to(dtype)

    s = dict(case)
    if case["op"] == "norm":
        r, c, wd = case["rows"], case["cols"], DTYPES[case["wdtype"]]
        s.update(x=randn(r, c, scale=1.5, mean=0.3), w=randn(c, scale=0.2, mean=1.0, dtype=wd), b=randn(c, scale=0.1, dtype=wd))
        leaves = ["x", "w", "b"]
        if case["train"]:
            s["dy"] = randn(r, c)
    elif case["op"] == "linear":
        m, n, k = case["m"], case["n"], case["k"]
        s.update(x=randn(m, k), w=randn(n, k, scale=k ** -0.5), b=randn(n, scale=0.1) if case["bias"] else None,
                 r=randn(m, n) if case["residual"] else None)
        leaves = ["x", "w"] + (["b"] if case["bias"] else []) + (["r"] if case["residual"] else [])
        if case["train"]:
            s["dy"] = randn(m, n)
    else:
        b, t, d = case["b"], case["t"], case["d"]
        # forget gates mostly open (sigmoid(2) = 0.88), as trained recurrences have them
        s.update(x=randn(b, t, d), gate=randn(b, t, d, scale=1.5, mean=2.0), h0=randn(b, d, dtype=torch.float32),
                 lengths=torch.randint(0, t + 1, (b,), generator=g, device="cuda", dtype=torch.int32) if case["ragged"] else None)
        leaves = ["x", "gate", "h0"]
        if case["train"]:
            s.update(dy=randn(b, t, d), dh=randn(b, d, dtype=torch.float32))
    s["leaves"] = leaves
    if case["train"]:
        for name in leaves:
            s[name].requires_grad_()
    return s


# ------------------------------------------------------------------------------------- plain operators
def _act(p, act):
    if act == "leaky":
        return torch.where(p > 0, p, SLOPE * p)
    if act == "sigmoid":
        return 1 / (1 + torch.exp(-p))
    if act == "gelu":
        return 0.5 * p * (1 + torch.erf(p * 0.5 ** 0.5))
    if act == "silu":
        return p / (1 + torch.exp(-p))
    return p


def _act_grad(p, act):
    if act == "leaky":
        return torch.where(p > 0, 1.0, SLOPE)
    if act == "sigmoid":
        y = 1 / (1 + torch.exp(-p))
        return y * (1 - y)
    if act == "gelu":
        return 0.5 * (1 + torch.erf(p * 0.5 ** 0.5)) + p * torch.exp(-0.5 * p * p) * (0.5 / math.pi) ** 0.5
    if act == "silu":
        y = 1 / (1 + torch.exp(-p))
        return y * (1 + p * (1 - y))
    return torch.ones_like(p)


def _plain_norm(s):
    x, w, b = s["x"].float(), s["w"].float(), s["b"].float()
    xc = x - x.mean(1, keepdim=True)
    rstd = 1 / torch.sqrt((xc * xc).mean(1, keepdim=True) + EPS)
    xhat = xc * rstd
    out = {"y": (xhat * w + b).to(s["x"].dtype)}
    if s["train"]:
        dy = s["dy"].float()
        g = dy * w
        dx = rstd * (g - g.mean(1, keepdim=True) - xhat * (g * xhat).mean(1, keepdim=True))
        out.update(dx=dx.to(s["x"].dtype), dw=(dy * xhat).sum(0).to(s["w"].dtype), db=dy.sum(0).to(s["b"].dtype))
    return out


def _plain_linear(s):
    x, w, dt = s["x"].float(), s["w"].float(), s["x"].dtype
    p = x @ w.t()
    if s["b"] is not None:
        p = p + s["b"].float()
    y = _act(p, s["act"])
    if s["r"] is not None:
        y = y + s["r"].float()
    out = {"y": y.to(dt)}
    if s["train"]:
        dp = s["dy"].float() * _act_grad(p, s["act"])
        out.update(dx=(dp @ w).to(dt), dw=(dp.t() @ x).to(dt))
        if s["b"] is not None:
            out["db"] = dp.sum(0).to(dt)
        if s["r"] is not None:
            out["dr"] = s["dy"]
    return out


def _recur(a, b):
    """h_t = a_t h_{t-1} + b_t along dim 1 by doubling: after the round of stride s every step holds 2s terms."""
    s = 1
    while s < a.shape[1]:
        b = torch.cat([b[:, :s], b[:, s:] + a[:, s:] * b[:, :-s]], 1)
        a = torch.cat([a[:, :s], a[:, s:] * a[:, :-s]], 1)
        s *= 2
    return b


def _plain_scan(s):
    x, gate, h0, dt = s["x"].float(), s["gate"].float(), s["h0"], s["x"].dtype
    f, i = 1 / (1 + torch.exp(-gate)), 1 / (1 + torch.exp(gate))
    if s["lengths"] is not None:  # steps behind a sequence's end hold the state
        live = (torch.arange(x.shape[1], device=x.device)[None] < s["lengths"][:, None])[..., None]
        f, i = torch.where(live, f, 1.0), torch.where(live, i, 0.0)
    b = i * x
    h = _recur(f, torch.cat([b[:, :1] + f[:, :1] * h0[:, None], b[:, 1:]], 1))
    y = h if s["lengths"] is None else torch.where(live, h, 0.0)
    out = {"y": y.to(dt), "h": h[:, -1].clone()}
    if s["train"]:
        dy = s["dy"].float()
        if s["lengths"] is not None:
            dy = torch.where(live, dy, 0.0)
        dy = torch.cat([dy[:, :-1], dy[:, -1:] + s["dh"][:, None]], 1)
        later = torch.cat([f[:, 1:], torch.zeros_like(f[:, :1])], 1)
        dh = _recur(later.flip(1), dy.flip(1)).flip(1)
        before = torch.cat([h0[:, None], h[:, :-1]], 1)
        out.update(dx=(i * dh).to(dt), dgate=(dh * (before - x) * f * i).to(dt), dh0=f[:, 0] * dh[:, 0])
    return out


# ------------------------------------------------------------------------------------------------- run
def _own(s):
    from vae_amd import layers
    if s["op"] == "norm":
        y = layers.layer_norm(s["x"], s["w"], s["b"], EPS)
        if not s["train"]:
            return {"y": y}
        dx, dw, db = torch.autograd.grad(y, [s["x"], s["w"], s["b"]], s["dy"])
        return {"y": y, "dx": dx, "dw": dw, "db": db}
    if s["op"] == "linear":
        y = layers.linear(s["x"], s["w"], s["b"], act=s["act"], slope=SLOPE, residual=s["r"])
        if not s["train"]:
            return {"y": y}
        grads = torch.autograd.grad(y, [s[k] for k in s["leaves"]], s["dy"])
        return {"y": y, **{"d" + k: v for k, v in zip(s["leaves"], grads)}}
    y, h = layers.gated_scan(s["x"], s["gate"], s["h0"], lengths=s["lengths"])
    if not s["train"]:
        return {"y": y, "h": h}
    dx, dgate, dh0 = torch.autograd.grad([y, h], [s["x"], s["gate"], s["h0"]], [s["dy"], s["dh"]])
    return {"y": y, "h": h, "dx": dx, "dgate": dgate, "dh0": dh0}


def run(state):
    if own:
        return _own(state)
    with torch.no_grad():
        return {"norm": _plain_norm, "linear": _plain_linear, "scan": _plain_scan}[state["op"]](state)


def work(case):
    e = ESIZE[case["dtype"]]
    if case["op"] == "norm":
        n, p = case["rows"] * case["cols"], case["cols"] * ESIZE[case["wdtype"]]
        return {"bytes": (4 * n * e + 4 * p) if case["train"] else (2 * n * e + 2 * p), "flops": n * (20 if case["train"] else 8)}
    if case["op"] == "linear":
        m, n, k = case["m"], case["n"], case["k"]
        once = m * k + n * k + m * n * (2 if case["residual"] else 1) + (n if case["bias"] else 0)
        back = m * n + m * k + n * k + (n if case["bias"] else 0)
        return {"bytes": (once + (back if case["train"] else 0)) * e, "flops": 2 * m * n * k * (3 if case["train"] else 1)}
    n, st = case["b"] * case["t"] * case["d"], case["b"] * case["d"] * 4
    return {"bytes": (6 * n * e + 4 * st) if case["train"] else (3 * n * e + 2 * st), "flops": n * (30 if case["train"] else 10)}


# ----------------------------------------------------------------------------------------------- exact
def _exact_norm(s):
    x, w, b = s["x"].double(), s["w"].double(), s["b"].double()
    c = x.shape[1]
    mean = x.sum(1) / c
    var = (x * x).sum(1) / c - mean * mean
    inv = (var + EPS).rsqrt()
    out = {"y": (x - mean[:, None]) * inv[:, None] * w[None] + b[None]}
    if s["train"]:
        dy = s["dy"].double()
        a = dy * w
        # d/dx of (x - mean) inv, written with the row's moments
        p, q = a.sum(1) / c, (a * x).sum(1) / c
        k = (q - p * mean) * inv ** 3
        out["dx"] = a * inv[:, None] - x * k[:, None] + (mean * k - p * inv)[:, None]
        out["dw"] = torch.einsum("rc,rc,r->c", dy, x, inv) - torch.einsum("rc,r->c", dy, mean * inv)
        out["db"] = dy.sum(0)
    return out


def _exact_linear(s):
    x, w = s["x"].double(), s["w"].double()
    p = torch.mm(x, w.t().contiguous())
    if s["b"] is not None:
        p += s["b"].double()[None]
    p.requires_grad_()
    with torch.enable_grad():
        act = s["act"]
        if act == "none":
            y = p * 1.0
        elif act == "leaky":
            y = p.clamp(min=0) + SLOPE * p.clamp(max=0)
        elif act == "sigmoid":
            y = torch.sigmoid(p)
        elif act == "gelu":
            y = p * torch.special.ndtr(p)
        else:
            y = p * torch.sigmoid(p)
    out = {"y": y.detach() if s["r"] is None else y.detach() + s["r"].double()}
    if s["train"]:
        (dp,) = torch.autograd.grad(y, p, s["dy"].double())
        out["dx"], out["dw"] = torch.mm(dp, w), torch.mm(dp.t().contiguous(), x)
        if s["b"] is not None:
            out["db"] = dp.sum(0)
        if s["r"] is not None:
            out["dr"] = s["dy"].double()
    return out


def _exact_scan(s):
    """Step by step, time in front so that a step is one contiguous slice."""
    x, gate = s["x"].double().transpose(0, 1).contiguous(), s["gate"].double().transpose(0, 1).contiguous()
    f, steps = torch.sigmoid(gate), x.shape[0]
    live = None
    if s["lengths"] is not None:
        live = (torch.arange(steps, device=x.device)[:, None] < s["lengths"][None, :])[..., None]
        f = f.masked_fill(~live, 1.0)
    h = torch.empty(steps + 1, *x.shape[1:], dtype=torch.float64, device=x.device)
    h[0] = s["h0"].double()
    for t in range(steps):
        torch.lerp(x[t], h[t], f[t], out=h[t + 1])  # x + f (h - x)
    y = h[1:] if live is None else h[1:].masked_fill(~live, 0.0)
    out = {"y": y.transpose(0, 1), "h": h[steps]}
    if s["train"]:
        dy = s["dy"].double().transpose(0, 1).contiguous()
        if live is not None:
            dy = dy.masked_fill(~live, 0.0)
        dh = torch.empty_like(dy)
        carry = s["dh"].double()
        for t in range(steps - 1, -1, -1):
            torch.add(dy[t], carry, out=dh[t])
            carry = dh[t] * f[t]
        keep = torch.sigmoid(-gate) if live is None else torch.sigmoid(-gate).masked_fill(~live, 0.0)
        out["dx"] = (dh * keep).transpose(0, 1)
        out["dgate"] = (dh * (h[:-1] - x) * f * keep).transpose(0, 1)
        out["dh0"] = carry
    return out


def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        return {"norm": _exact_norm, "linear": _exact_linear, "scan": _exact_scan}[case["op"]](s)
