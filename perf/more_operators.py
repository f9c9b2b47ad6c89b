"""Cases of a decoder layer's operators between its attention calls: normalisation, linear layers with what follows
them, and the gated feed-forward block.

Operators (`op`):
  norm    `layers.layer_norm`: layer norm over the last axis
  linear  `layers.linear`: product with a weight, bias, activation and residual
  gated   `layers.gated_feed_forward`: (act(x Wg^T) * (x Wu^T)) Wd^T, with or without residual

`train` false is a forward pass (scoring, prompts, single tokens); true is a forward and a backward pass, whose gradients
are returned.  With `own` false `run` computes the plain form in torch operations, else it calls the package.
"""
import importlib
import math

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def _norm(name, train, n, d, dtype, params="same"):
    return dict(name=name, op="norm", train=train, n=n, d=d, dtype=dtype, params=params)


def _linear(name, train, n, k, m, dtype, act="none", bias=True, residual=False, apart=0):
    return dict(name=name, op="linear", train=train, n=n, k=k, m=m, dtype=dtype, act=act, bias=bias, residual=residual, apart=apart)


def _gated(name, train, n, d, f, dtype, act="silu", residual=True):
    return dict(name=name, op="gated", train=train, n=n, d=d, f=f, dtype=dtype, act=act, residual=residual)


def listed():
    return [
        # a short prompt through one norm of the 768-wide model of bench_ttt.py: launches and latency
        _norm("norm_score_200", False, 200, 768, "bf16"),
        # that model in training, 8 x 2048 tokens
        _norm("norm_train_16384", True, 16384, 768, "bf16"),
        # wide rows, an odd number of them, parameters kept in float32
        _norm("norm_train_wide", True, 8195, 4096, "fp16", "float"),
        # fp32 with a width that no vector load divides: gradient checks and debugging
        _norm("norm_fp32_odd", True, 1031, 777, "fp32"),
        # the projection of Q, K and V of one token
        _linear("linear_token", False, 1, 768, 2304, "bf16"),
        # the first layer of a GELU MLP in training, 8 x 2048 tokens
        _linear("linear_train_16384", True, 16384, 768, 2048, "bf16", "gelu"),
        # wide rows that are a slice of another projection's result, an odd number of tokens, bias and residual
        _linear("linear_train_wide", True, 4099, 2048, 5504, "fp16", "none", True, True, 64),
        # fp32, sizes that fit no tile
        _linear("linear_fp32", True, 333, 200, 515, "fp32", "gelu_tanh"),
        # one token through a block
        _gated("gated_token", False, 1, 2048, 5504, "bf16"),
        # the 768-wide model with a gated block in training
        _gated("gated_train_16384", True, 16384, 768, 2048, "bf16"),
        # wider, an odd number of tokens
        _gated("gated_train_wide", True, 4099, 2048, 5504, "fp16"),
        # fp32, sizes that fit no tile
        _gated("gated_fp32", True, 201, 136, 345, "fp32", "gelu", False),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _width(rng, lo, hi):
    """Mostly a multiple of eight, as models have them, else any number."""
    return 8 * _log_int(rng, max(1, lo // 8), hi // 8) if rng.random() < 0.8 else _log_int(rng, lo, hi)


def draw(rng):
    op = rng.choice(("norm", "linear", "linear", "gated", "gated"))
    train = rng.random() < 0.6
    dtype = rng.choice(("bf16", "bf16", "fp16", "fp32"))
    act = rng.choice(("silu", "gelu", "gelu_tanh"))
    if op == "norm":
        d = _width(rng, 8, 8192)
        most = min(16384, (30000000 if dtype != "fp32" else 16000000) // d)
        return dict(op=op, train=train, n=_log_int(rng, 1, most), d=d, dtype=dtype, params=rng.choice(("same", "same", "float", "none")))
    residual = rng.random() < 0.5
    if op == "linear":
        hi = (700, 400, 900) if dtype == "fp32" else (8000, 2048, 5504)
        return dict(op=op, train=train, n=_log_int(rng, 1, hi[0]), k=_width(rng, 16, hi[1]), m=_width(rng, 16, hi[2]), dtype=dtype,
                    act=rng.choice(("none", act)), bias=rng.random() < 0.5, residual=residual, apart=rng.choice((0, 0, 8, 64)))
    hi = (300, 256, 600) if dtype == "fp32" else (4099, 2048, 5504)
    return dict(op=op, train=train, n=_log_int(rng, 1, hi[0]), d=_width(rng, 16, hi[1]), f=_width(rng, 16, hi[2]), dtype=dtype,
                act=act, residual=residual)


def work(case):
    size = 4 if case["dtype"] == "fp32" else 2
    n = case["n"]
    if case["op"] == "norm":
        d = case["d"]
        # forward: x in, y out; backward: g in, gx out beside them
        return {"bytes": n * d * size * (4 if case["train"] else 2), "flops": n * d * (24 if case["train"] else 8)}
    if case["op"] == "linear":
        k, m = case["k"], case["m"]
        elements = n * k + m * k + n * m * (2 if case["residual"] else 1)     # x, w; y, residual
        if case["train"]:
            elements += n * k + m * k + n * m                                 # gx, gw; g
        return {"bytes": elements * size, "flops": (6 if case["train"] else 2) * n * k * m}
    d, f = case["d"], case["f"]
    elements = 3 * d * f + n * d * (3 if case["residual"] else 2)             # the weights; x, y, residual
    if case["train"]:
        elements += 3 * d * f + 2 * n * d                                     # the weights' gradients; g, gx
    return {"bytes": elements * size, "flops": (18 if case["train"] else 6) * n * d * f}


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = _DTYPES[case["dtype"]]

    def randn(*shape, std=1.0, mean=0.0, dtype=dt):
        return (torch.randn(*shape, generator=g, device="cuda") * std + mean).to(dtype)

    s, n = dict(case=case), case["n"]
    if case["op"] == "norm":
        d = case["d"]
        # a residual stream: rows of different size around means that are not 0
        spread = torch.rand(n, 1, generator=g, device="cuda") * 3 + 0.3
        centre = torch.randn(n, 1, generator=g, device="cuda")
        s["x"] = (torch.randn(n, d, generator=g, device="cuda") * spread + centre).to(dt)
        pt = torch.float32 if case["params"] == "float" else dt
        s["w"] = randn(d, std=0.2, mean=1.0, dtype=pt) if case["params"] != "none" else None
        s["b"] = randn(d, std=0.2, dtype=pt) if case["params"] != "none" else None
        s["g"] = randn(n, d)
    elif case["op"] == "linear":
        k, m = case["k"], case["m"]
        wide = randn(n, k + case["apart"])                       # rows behind a norm
        s["x"] = wide[:, :k]
        s["w"] = randn(m, k, std=1.5 / math.sqrt(k))
        s["b"] = randn(m, std=0.3) if case["bias"] else None
        s["r"] = randn(n, m) if case["residual"] else None
        s["g"] = randn(n, m)
    else:
        d, f = case["d"], case["f"]
        s["x"] = randn(n, d)
        s["wg"], s["wu"] = randn(f, d, std=1.5 / math.sqrt(d)), randn(f, d, std=1.5 / math.sqrt(d))
        s["wd"] = randn(d, f, std=1.5 / math.sqrt(f))
        s["r"] = randn(n, d) if case["residual"] else None
        s["g"] = randn(n, d)
    return s


# ---- plain forms --------------------------------------------------------------------------------

def _act(z, kind):
    """(activation, its derivative)"""
    if kind == "none":
        return z, torch.ones_like(z)
    if kind == "gelu":
        below = 0.5 * torch.erfc(z * -math.sqrt(0.5))
        return z * below, below + z * torch.exp(-0.5 * z * z) * (1.0 / math.sqrt(2 * math.pi))
    if kind == "silu":
        u, du = z, torch.ones_like(z)
    else:      # gelu_tanh: 0.5 (1 + tanh(u / 2)) is the logistic function of u
        u = 2 * math.sqrt(2 / math.pi) * (z + 0.044715 * z * z * z)
        du = 2 * math.sqrt(2 / math.pi) * (1 + 3 * 0.044715 * z * z)
    e = torch.exp(-u.abs())
    share = torch.where(u >= 0, 1 / (1 + e), e / (1 + e))
    return z * share, share + z * du * e / ((1 + e) * (1 + e))


def _plain_norm(s):
    dt, x = s["x"].dtype, s["x"].float()
    w = s["w"].float() if s["w"] is not None else torch.ones(x.shape[1], device="cuda")
    centred = x - x.mean(-1, keepdim=True)
    r = 1 / torch.sqrt((centred * centred).mean(-1, keepdim=True) + 1e-5)
    unit = centred * r
    y = unit * w
    if s["b"] is not None:
        y = y + s["b"].float()
    if not s["case"]["train"]:
        return y.to(dt)
    g = s["g"].float()
    gu = g * w
    gx = r * (gu - gu.mean(-1, keepdim=True) - unit * (gu * unit).mean(-1, keepdim=True))
    if s["w"] is None:
        return y.to(dt), gx.to(dt)
    return (y.to(dt), gx.to(dt), (g * unit).sum(0, dtype=torch.float64).to(s["w"].dtype), g.sum(0, dtype=torch.float64).to(s["b"].dtype))


def _plain_linear(s):
    dt, x, w = s["x"].dtype, s["x"].float(), s["w"].float()
    z = x @ w.T
    if s["b"] is not None:
        z = z + s["b"].float()
    y, slope = _act(z, s["case"]["act"])
    if s["r"] is not None:
        y = y + s["r"].float()
    if not s["case"]["train"]:
        return y.to(dt)
    gz = s["g"].float() * slope
    out = [y.to(dt), (gz @ w).to(dt), (gz.T @ x).to(dt)]
    if s["b"] is not None:
        out.append(gz.sum(0, dtype=torch.float64).to(dt))
    if s["r"] is not None:
        out.append(s["g"])
    return tuple(out)


def _plain_gated(s):
    dt, x = s["x"].dtype, s["x"].float()
    wg, wu, wd = s["wg"].float(), s["wu"].float(), s["wd"].float()
    up = x @ wu.T
    a, slope = _act(x @ wg.T, s["case"]["act"])
    h = a * up
    y = h @ wd.T
    if s["r"] is not None:
        y = y + s["r"].float()
    if not s["case"]["train"]:
        return y.to(dt)
    g = s["g"].float()
    gh = g @ wd
    gg, gu = gh * up * slope, gh * a
    out = [y.to(dt), (gg @ wg + gu @ wu).to(dt), (gg.T @ x).to(dt), (gu.T @ x).to(dt), (g.T @ h).to(dt)]
    if s["r"] is not None:
        out.append(s["g"])
    return tuple(out)


# ---- one pass -----------------------------------------------------------------------------------

def _leaves(s, names):
    return {name: None if s[name] is None else s[name].detach().requires_grad_(s["case"]["train"]) for name in names}


def _pass(s, names, call):
    t = _leaves(s, names)
    out = call(t)
    if not s["case"]["train"]:
        return out
    return (out.detach(), *torch.autograd.grad(out, [v for v in t.values() if v is not None], s["g"]))


def _kind(case):
    return None if case["act"] == "none" else case["act"]


def _own_norm(s):
    layers = importlib.import_module("610sample_b200.layers")
    return _pass(s, ("x", "w", "b"), lambda t: layers.layer_norm(t["x"], t["w"], t["b"]))


def _own_linear(s):
    layers = importlib.import_module("610sample_b200.layers")
    return _pass(s, ("x", "w", "b", "r"), lambda t: layers.linear(t["x"], t["w"], t["b"], activation=_kind(s["case"]), residual=t["r"]))


def _own_gated(s):
    layers = importlib.import_module("610sample_b200.layers")
    return _pass(s, ("x", "wg", "wu", "wd", "r"), lambda t: layers.gated_feed_forward(
        t["x"], t["wg"], t["wu"], t["wd"], activation=_kind(s["case"]), residual=t["r"]))


def run(state):
    op = state["case"]["op"]
    if own:
        return {"norm": _own_norm, "linear": _own_linear, "gated": _own_gated}[op](state)
    return {"norm": _plain_norm, "linear": _plain_linear, "gated": _plain_gated}[op](state)


# ---- the operators' definitions in 64 bits --------------------------------------------------------

_CURVES = {
    None: lambda z: z,
    "none": lambda z: z,
    "silu": lambda z: z * torch.sigmoid(z),
    "gelu": lambda z: 0.5 * z * torch.erfc(-z / 2 ** 0.5),
    "gelu_tanh": lambda z: z * torch.sigmoid((8 / math.pi) ** 0.5 * (z + 0.044715 * z ** 3)),
}


def _define_norm(t, case):
    x = t["x"]
    var, mean = torch.var_mean(x, -1, correction=0, keepdim=True)
    y = (x - mean) * torch.rsqrt(var + 1e-5)
    return y if t["w"] is None else y * t["w"] + t["b"]


def _define_linear(t, case):
    z = torch.matmul(t["x"], t["w"].t())
    y = _CURVES[case["act"]](z if t["b"] is None else z + t["b"])
    return y if t["r"] is None else t["r"] + y


def _define_gated(t, case):
    inner = _CURVES[case["act"]](torch.matmul(t["x"], t["wg"].t())) * torch.matmul(t["x"], t["wu"].t())
    y = torch.matmul(inner, t["wd"].t())
    return y if t["r"] is None else t["r"] + y


def exact(case, seed):
    state = prepare(case, seed)
    define, names = {"norm": (_define_norm, ("x", "w", "b")), "linear": (_define_linear, ("x", "w", "b", "r")),
                     "gated": (_define_gated, ("x", "wg", "wu", "wd", "r"))}[case["op"]]
    t = {name: None if state[name] is None else state[name].double().requires_grad_(case["train"]) for name in names}
    y = define(t, case)
    if not case["train"]:
        return y
    return (y.detach(), *torch.autograd.grad(y, [v for v in t.values() if v is not None], state["g"].double()))
