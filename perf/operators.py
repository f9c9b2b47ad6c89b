"""Cases of the packed-batch operators: what training and scoring on batches of documents of different
lengths, laid end to end without padding, spends its time on outside the model's own matrix products.

Operators (`op`):
  attn   `packed.packed_attention`: causal attention within each document, grouped key/value heads
  loss   `loss.linear_cross_entropy`: head projection and cross entropy without kept logits
  rope   `packed.packed_qk_norm_rope`: norm of Q and K per head and rotation by per-token positions

`train` false is a forward pass (scoring, prompts); true is a forward and a backward pass, whose gradients
are returned.  With `own` false `run` computes the plain form in torch operations, else it calls the package.
"""
import importlib
import math
import random

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def _attn(name, train, n_tok, n_seq, tail, Hq, Hkv, D, window, dtype):
    return dict(name=name, op="attn", train=train, n_tok=n_tok, n_seq=n_seq, tail=tail, Hq=Hq, Hkv=Hkv, D=D,
                window=window, dtype=dtype, cut=n_tok + 7 * n_seq)


def _loss(name, train, n, d, V, dtype, reduction="mean"):
    return dict(name=name, op="loss", train=train, n=n, d=d, V=V, dtype=dtype, reduction=reduction)


def _rope(name, train, n_tok, Hq, Hkv, D, axes, dtype):
    return dict(name=name, op="rope", train=train, n_tok=n_tok, Hq=Hq, Hkv=Hkv, D=D, axes=axes, dtype=dtype)


def listed():
    return [
        # a handful of short texts scored together: launches and latency
        _attn("attn_score_200", False, 200, 3, 0, 12, 12, 64, 0, "bf16"),
        # one layer of the 12-head model of bench_ttt.py, 8 x 2048 tokens as documents of all lengths
        _attn("attn_train_16384_h12", True, 16384, 19, 0, 12, 12, 64, 0, "bf16"),
        # grouped heads of 128, half-filled last documents and unused rows behind them
        _attn("attn_train_8192_gqa", True, 8192, 7, 113, 32, 8, 128, 0, "bf16"),
        # one long prompt
        _attn("attn_prompt_32768", False, 32768, 1, 0, 16, 4, 128, 0, "fp16"),
        # fp32 with a sliding window and an odd number of rows: gradient checks and debugging
        _attn("attn_fp32_window", True, 1031, 5, 6, 6, 2, 80, 100, "fp32"),
        # the loss of a few candidate continuations, one value per token
        _loss("loss_score_37", False, 37, 768, 32000, "bf16", "none"),
        # the head of bench_ttt.py in training: 8 x 2048 tokens
        _loss("loss_train_16384", True, 16384, 768, 32000, "bf16"),
        # a larger vocabulary with an odd size, wider rows, an odd number of tokens (fp16 trains on a scaled loss)
        _loss("loss_train_wide", True, 4099, 2048, 100003, "fp16", "sum"),
        # fp32, sizes that fit no tile
        _loss("loss_fp32", True, 333, 200, 5003, "fp32", "sum"),
        # a short prompt's Q and K
        _rope("rope_score_200", False, 200, 12, 12, 64, 1, "bf16"),
        # the 12-head model in training
        _rope("rope_train_16384", True, 16384, 12, 12, 64, 1, "bf16"),
        # video patches: time, height and width share the pairs of a head
        _rope("rope_train_video", True, 30011, 32, 8, 128, 3, "fp16"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("attn", "attn", "loss", "loss", "rope"))
    train = rng.random() < 0.6
    dtype = rng.choice(("bf16", "bf16", "fp16", "fp32"))
    if op == "attn":
        D = rng.choice((32, 64, 64, 80, 96, 128, 128))
        Hkv = rng.choice((1, 2, 4, 6, 8))
        Hq = Hkv * rng.choice((1, 1, 2, 4, 5))
        n_tok = _log_int(rng, 1, 1500 if dtype == "fp32" else 20000)
        n_seq = min(_log_int(rng, 1, 40), n_tok)
        tail = rng.choice((0, 0, rng.randrange(0, 1 + n_tok // 8)))
        window = rng.choice((0, 0, _log_int(rng, 1, 4096)))
        return dict(op=op, train=train, n_tok=n_tok, n_seq=n_seq, tail=tail, Hq=Hq, Hkv=Hkv, D=D, window=window,
                    dtype=dtype, cut=rng.randrange(1 << 30))
    if op == "loss":
        if dtype == "fp32":
            n, d, V = _log_int(rng, 1, 700), _log_int(rng, 8, 400), _log_int(rng, 2, 6000)
        else:
            n, d, V = _log_int(rng, 1, 8000), 8 * _log_int(rng, 4, 256), _log_int(rng, 2, 100003)
        return dict(op=op, train=train, n=n, d=d, V=V, dtype=dtype,
                    reduction=rng.choice(("sum", "none") if dtype == "fp16" else ("mean", "sum", "none")))
    Hkv = rng.choice((1, 2, 4, 6, 8, 12))
    return dict(op=op, train=train, n_tok=_log_int(rng, 1, 16000 if dtype == "fp32" else 30000), Hq=Hkv * rng.choice((1, 2, 4)),
                Hkv=Hkv, D=rng.choice((32, 40, 64, 80, 96, 128)), axes=rng.choice((1, 1, 2, 3)), dtype=dtype)


def _lengths(case):
    """Documents of all lengths, none to most of the batch, that fill all rows but the last `tail`."""
    rng = random.Random(case["cut"])
    total = case["n_tok"] - case["tail"]
    weights = [rng.expovariate(1.0) ** 1.5 + 1e-3 for _ in range(case["n_seq"])]
    scale = total / sum(weights)
    lens = [int(w * scale) for w in weights]
    lens[rng.randrange(len(lens))] += total - sum(lens)
    return lens


def _sections(case):
    pairs, axes = case["D"] // 2, case["axes"]
    first = pairs // (axes + 1) if axes > 1 else pairs      # the first axis (time) gets the smaller share
    sections = [first]
    while len(sections) < axes:
        sections.append((pairs - sum(sections)) // (axes - len(sections)))
    return tuple(sections)


def _pairs(case):
    w = case["window"] or case["n_tok"]
    total = 0
    for n in _lengths(case):
        full = min(n, w)
        total += full * (full + 1) // 2 + (n - full) * w
    return total


def work(case):
    size = 4 if case["dtype"] == "fp32" else 2
    if case["op"] == "attn":
        n, D, Hq, Hkv = case["n_tok"], case["D"], case["Hq"], case["Hkv"]
        tensors = n * D * (2 * Hq + 2 * Hkv)                          # q, O; k, v
        if case["train"]:
            tensors += n * D * (2 * Hq + 2 * Hkv)                     # dO, dq; dk, dv
        return {"bytes": tensors * size, "flops": (14 if case["train"] else 4) * D * Hq * _pairs(case)}
    if case["op"] == "loss":
        n, d, V = case["n"], case["d"], case["V"]
        rows = (n + V) * d * size
        return {"bytes": rows * (2 if case["train"] else 1) + 8 * n, "flops": (6 if case["train"] else 2) * n * d * V}
    n, D, H = case["n_tok"], case["D"], case["Hq"] + case["Hkv"]
    table = n * (case["axes"] * 4)
    # forward: x in, y out; backward: x and g in, gx out
    passes = 2 if not case["train"] else 5
    return {"bytes": n * H * D * size * passes + table, "flops": n * H * D * (8 if not case["train"] else 28)}


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = _DTYPES[case["dtype"]]

    def randn(*shape, std=1.0, mean=0.0):
        return (torch.randn(*shape, generator=g, device="cuda") * std + mean).to(dt)

    s = dict(case=case)
    if case["op"] == "attn":
        n, D, Hq, Hkv = case["n_tok"], case["D"], case["Hq"], case["Hkv"]
        # one projection's result; q and k have been normed per head, so scores have a spread of about 2
        qkv = randn(n, Hq + 2 * Hkv, D)
        qkv[:, :Hq + Hkv] *= 1.4
        s["q"], s["k"], s["v"] = qkv[:, :Hq], qkv[:, Hq:Hq + Hkv], qkv[:, Hq + Hkv:]
        s["g"] = randn(n, Hq, D)
        s["lens"] = _lengths(case)
        offsets = [0]
        for length in s["lens"]:
            offsets.append(offsets[-1] + length)
        s["cu_seqlens"] = torch.tensor(offsets, dtype=torch.int32, device="cuda")
        s["window"] = case["window"] or None
        if own:      # made once per batch and shared by all layers
            s["plan"] = importlib.import_module("610sample_b200.packed").packed_plan(s["cu_seqlens"], n)
    elif case["op"] == "loss":
        n, d, V = case["n"], case["d"], case["V"]
        s["x"] = randn(n, d)                                     # rows behind a final norm
        s["w"] = randn(V, d, std=2.5 / math.sqrt(d))             # logits with a spread of 2.5
        y = torch.randint(0, V, (n,), generator=g, device="cuda")
        skip = torch.rand(n, generator=g, device="cuda") < 0.06  # the last token of a document predicts nothing
        s["y"] = torch.where(skip, torch.full_like(y, -100), y)
        if n < 8:
            s["y"][0] = y[0]
        s["g"] = torch.rand(n, generator=g, device="cuda") + 0.5
    else:
        n, D, Hq, Hkv, axes = case["n_tok"], case["D"], case["Hq"], case["Hkv"], case["axes"]
        qkv = randn(n, Hq + 2 * Hkv, D, std=1.7)
        s["q"], s["k"] = qkv[:, :Hq], qkv[:, Hq:Hq + Hkv]
        s["qw"], s["kw"] = randn(D, std=0.1, mean=1.0), randn(D, std=0.1, mean=1.0)
        s["sections"] = _sections(case)
        t = torch.arange(n, device="cuda")
        if axes == 1:        # documents of 1000 or so, each starting from position 0
            start = torch.rand(n, generator=g, device="cuda") < 0.001
            first = torch.cummax(torch.where(start, t, torch.zeros_like(t)), 0).values
            s["positions"] = (t - first).to(torch.int32)
        else:                # patches of frames of 24 x 40
            grid = [t // 960, (t // 40) % 24, t % 40]
            s["positions"] = torch.stack(grid[:axes]).to(torch.int32)
        rows = int(max(n, 64))
        inv = 10000.0 ** (-torch.arange(0, D, 2, device="cuda", dtype=torch.float64) / D)
        ang = torch.outer(torch.arange(rows, device="cuda", dtype=torch.float64), inv)
        s["freqs"] = torch.stack([ang.cos(), ang.sin()], dim=-1).float().contiguous()
        s["gq"], s["gk"] = randn(n, Hq, D), randn(n, Hkv, D)
    return s


# ---- plain forms --------------------------------------------------------------------------------

def _visible(i0, i1, n_keys, window, device):
    i = torch.arange(i0, i1, device=device)[:, None]
    j = torch.arange(n_keys, device=device)[None, :]
    seen = j <= i
    return seen if window is None else seen & (i < j + window)


def _plain_attn(s):
    case = s["case"]
    n, D, Hq, Hkv = case["n_tok"], case["D"], case["Hq"], case["Hkv"]
    group, scale, dt = Hq // Hkv, 1.0 / math.sqrt(D), s["q"].dtype
    out = torch.zeros(n, Hq, D, device="cuda")
    if case["train"]:
        dq, dk, dv = torch.zeros(n, Hq, D, device="cuda"), torch.zeros(n, Hkv, D, device="cuda"), torch.zeros(n, Hkv, D, device="cuda")
    a = 0
    for length in s["lens"]:
        b = a + length
        for h in range(Hkv if length else 0):
            heads = slice(h * group, (h + 1) * group)
            k, v = s["k"][a:b, h].float(), s["v"][a:b, h].float()
            step = max(64, min(length, (1 << 28) // (group * length)))
            for i0 in range(0, length, step):
                i1 = min(i0 + step, length)
                q = s["q"][a + i0:a + i1, heads].float().transpose(0, 1)
                seen = _visible(i0, i1, i1, s["window"], q.device)
                z = (q @ k[:i1].T) * scale
                z = torch.where(seen, z, torch.full_like(z, -math.inf))
                e = torch.exp(z - z.amax(-1, keepdim=True))
                p = e / e.sum(-1, keepdim=True)
                o = p @ v[:i1]
                out[a + i0:a + i1, heads] = o.transpose(0, 1)
                if case["train"]:
                    do = s["g"][a + i0:a + i1, heads].float().transpose(0, 1)
                    dp = do @ v[:i1].T
                    ds = p * (dp - (do * o).sum(-1, keepdim=True)) * scale
                    dq[a + i0:a + i1, heads] = (ds @ k[:i1]).transpose(0, 1)
                    dk[a:a + i1, h] += (ds.transpose(1, 2) @ q).sum(0)
                    dv[a:a + i1, h] += (p.transpose(1, 2) @ do).sum(0)
        a = b
    if not case["train"]:
        return out.to(dt)
    return out.to(dt), dq.to(dt), dk.to(dt), dv.to(dt)


def _plain_loss(s):
    case = s["case"]
    n, V, dt = case["n"], case["V"], s["x"].dtype
    w, y = s["w"].float(), s["y"]
    counted = y != -100
    losses = torch.zeros(n, device="cuda")
    if case["reduction"] == "none":
        coef = s["g"] * counted
    else:
        coef = counted.float() / (counted.sum() if case["reduction"] == "mean" else 1.0)
    if case["train"]:
        gx, gw = torch.empty(n, case["d"], device="cuda"), torch.zeros(V, case["d"], device="cuda")
    step = max(1, (1 << 29) // V)
    for i0 in range(0, n, step):
        x, yy, cc = s["x"][i0:i0 + step].float(), y[i0:i0 + step].clamp_min(0), counted[i0:i0 + step]
        z = x @ w.T
        top = z.amax(-1, keepdim=True)
        e = torch.exp(z - top)
        total = e.sum(-1, keepdim=True)
        loss = (top + torch.log(total))[:, 0] - z.gather(1, yy[:, None])[:, 0]
        losses[i0:i0 + step] = torch.where(cc, loss, torch.zeros_like(loss))
        if case["train"]:
            p = e / total
            p.scatter_add_(1, yy[:, None], torch.full((len(yy), 1), -1.0, device="cuda"))
            p *= coef[i0:i0 + step, None]
            gx[i0:i0 + step] = p @ w
            gw += p.T @ x
    if case["reduction"] == "mean":
        losses = losses.double().sum().float() / counted.sum()
    elif case["reduction"] == "sum":
        losses = losses.double().sum().float()
    return (losses, gx.to(dt), gw.to(dt)) if case["train"] else losses


def _angles(s):
    """cos and sin of every token and pair: the pair's axis names the position."""
    pos = s["positions"].long()
    pos = pos[None] if pos.dim() == 1 else pos
    axis = torch.repeat_interleave(torch.arange(len(s["sections"]), device="cuda"), torch.tensor(s["sections"], device="cuda"))
    pair = torch.arange(len(axis), device="cuda")
    return s["freqs"][pos[axis].T, pair[None, :]]            # [n_tok, pairs, 2]


def _plain_rope(s):
    case = s["case"]
    cs = _angles(s)
    c, sn = cs[:, None, :, 0], cs[:, None, :, 1]
    outs, grads, weights = [], [], []
    for x, w, g in ((s["q"], s["qw"], s["gq"]), (s["k"], s["kw"], s["gk"])):
        dt, xf, wf = x.dtype, x.float(), w.float()
        r = torch.rsqrt(xf.pow(2).mean(-1, keepdim=True) + 1e-6)
        y = xf * r * wf
        a, b = y[..., 0::2], y[..., 1::2]
        outs.append(torch.stack([a * c - b * sn, a * sn + b * c], -1).flatten(-2).to(dt))
        if case["train"]:
            gf = g.float()
            ga, gb = gf[..., 0::2], gf[..., 1::2]
            gy = torch.stack([ga * c + gb * sn, gb * c - ga * sn], -1).flatten(-2)
            gn = gy * wf
            grads.append((r * gn - xf * r.pow(3) * (gn * xf).mean(-1, keepdim=True)).to(dt))
            weights.append((gy * xf * r).sum((0, 1), dtype=torch.float64).to(dt))
    return tuple(outs + grads + weights)


# ---- one pass -----------------------------------------------------------------------------------

def _leaf(t):
    return t.detach().requires_grad_(True)


def _own_attn(s):
    packed = importlib.import_module("610sample_b200.packed")
    if not s["case"]["train"]:
        return packed.packed_attention(s["q"], s["k"], s["v"], s["plan"], s["window"])
    q, k, v = _leaf(s["q"]), _leaf(s["k"]), _leaf(s["v"])
    out = packed.packed_attention(q, k, v, s["plan"], s["window"])
    return (out.detach(), *torch.autograd.grad(out, (q, k, v), s["g"]))


def _own_loss(s):
    loss = importlib.import_module("610sample_b200.loss")
    reduction = s["case"]["reduction"]
    if not s["case"]["train"]:
        return loss.linear_cross_entropy(s["x"], s["w"], s["y"], reduction=reduction)
    x, w = _leaf(s["x"]), _leaf(s["w"])
    out = loss.linear_cross_entropy(x, w, s["y"], reduction=reduction)
    return (out.detach(), *torch.autograd.grad(out, (x, w), s["g"] if reduction == "none" else None))


def _own_rope(s):
    packed = importlib.import_module("610sample_b200.packed")
    if not s["case"]["train"]:
        return packed.packed_qk_norm_rope(s["q"], s["k"], s["qw"], s["kw"], s["freqs"], s["positions"], s["sections"])
    leaves = [_leaf(s[name]) for name in ("q", "k", "qw", "kw")]
    outs = packed.packed_qk_norm_rope(*leaves, s["freqs"], s["positions"], s["sections"])
    grads = torch.autograd.grad(outs, leaves, (s["gq"], s["gk"]))
    return (outs[0].detach(), outs[1].detach(), *grads)


def run(state):
    op = state["case"]["op"]
    if own:
        return {"attn": _own_attn, "loss": _own_loss, "rope": _own_rope}[op](state)
    return {"attn": _plain_attn, "loss": _plain_loss, "rope": _plain_rope}[op](state)


# ---- the operators' definitions in 64 bits --------------------------------------------------------

def _exact_attn(s):
    case = s["case"]
    D, group = case["D"], case["Hq"] // case["Hkv"]
    q, k, v = s["q"].double(), s["k"].double(), s["v"].double()
    dout = s["g"].double()
    out, dq, dk, dv = (torch.zeros_like(t) for t in (q, q, k, v))
    begin = 0
    for length in s["lens"]:
        rows = slice(begin, begin + length)
        begin += length
        for h in range(case["Hq"] if length else 0):
            kh, vh = k[rows, h // group], v[rows, h // group]
            block = max(1, (1 << 27) // length)
            for r0 in range(0, length, block):
                r1 = min(length, r0 + block)
                mine = slice(rows.start + r0, rows.start + r1)
                qh = q[mine, h]
                weight = torch.exp(_hide(qh @ kh[:r1].T / D ** 0.5, r0, case["window"]))
                total = weight.sum(1, keepdim=True)
                out[mine, h] = weight @ vh[:r1] / total
                if case["train"]:
                    prob = weight / total
                    gh = dout[mine, h]
                    dprob = gh @ vh[:r1].T
                    dscore = prob * (dprob - (prob * dprob).sum(1, keepdim=True))
                    dq[mine, h] = dscore @ kh[:r1] / D ** 0.5
                    dk[rows.start:rows.start + r1, h // group] += dscore.T @ qh / D ** 0.5
                    dv[rows.start:rows.start + r1, h // group] += prob.T @ gh
    return (out, dq, dk, dv) if case["train"] else out


def _hide(scores, r0, window):
    """Scores of rows r0, r0 + 1, ... with -inf at later keys and at keys that have left the window."""
    distance = torch.arange(r0, r0 + scores.shape[0], device=scores.device)[:, None] - torch.arange(scores.shape[1], device=scores.device)
    hidden = distance < 0
    if window:
        hidden |= distance >= window
    scores = scores - scores.masked_fill(hidden, -math.inf).amax(1, keepdim=True)
    return scores.masked_fill_(hidden, -math.inf)


def _exact_loss(s):
    case, x, w, y = s["case"], s["x"].double(), s["w"].double(), s["y"]
    keep = (y >= 0).double()
    share = keep / keep.sum() if case["reduction"] == "mean" else keep
    if case["reduction"] == "none":
        share = share * s["g"].double()
    nll, gx, gw = torch.empty(len(y), dtype=torch.float64, device="cuda"), torch.empty_like(x), torch.zeros_like(w)
    block = max(1, (1 << 28) // len(w))
    for rows in torch.arange(len(y), device="cuda").split(block):
        logp = torch.log_softmax(x[rows] @ w.T, -1)
        at = y[rows].clamp(min=0)
        local = torch.arange(len(rows), device="cuda")
        nll[rows] = -logp[local, at] * keep[rows]
        if case["train"]:
            d = logp.exp_()
            d[local, at] -= 1.0
            d *= share[rows, None]
            gx[rows] = d @ w
            gw.addmm_(d.T, x[rows])
    value = {"none": nll, "sum": nll.sum(), "mean": nll.sum() / keep.sum()}[case["reduction"]]
    return (value, gx, gw) if case["train"] else value


def _exact_rope(s):
    pos = s["positions"].reshape(-1, s["case"]["n_tok"]).long()
    turn, first = [], 0
    for axis, count in enumerate(s["sections"]):
        turn.append(s["freqs"].double()[pos[axis], first:first + count])
        first += count
    turn = torch.view_as_complex(torch.cat(turn, 1).contiguous())[:, None]
    outs, grads, weights = [], [], []
    for x, w, g in ((s["q"], s["qw"], s["gq"]), (s["k"], s["kw"], s["gk"])):
        x, w = x.double().requires_grad_(True), w.double().requires_grad_(True)
        unit = x / torch.sqrt((x * x).mean(-1, keepdim=True) + 1e-6)
        turned = torch.view_as_complex((unit * w).unflatten(-1, (-1, 2)).contiguous()) * turn
        out = torch.view_as_real(turned).flatten(-2)
        if s["case"]["train"]:
            gx, gw = torch.autograd.grad(out, (x, w), g.double())
            grads.append(gx)
            weights.append(gw)
        outs.append(out.detach())
    return tuple(outs + grads + weights)


def exact(case, seed):
    state = prepare(case, seed)
    return {"attn": _exact_attn, "loss": _exact_loss, "rope": _exact_rope}[case["op"]](state)
