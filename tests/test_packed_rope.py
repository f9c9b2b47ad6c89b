"""Norm and rotation of Q and K with per-token positions: refusals (CPU); results, gradients and the second derivative
against 64 bits with bounds derived from the roundings; and the packed operators together, as a layer and its loss
use them (GPU)."""
import ctypes
import importlib
import math
import os
import sys

import pytest
import torch

PKG_DIR = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "610sample_b200")


@pytest.fixture(scope="module")
def packed():
    if PKG_DIR not in sys.path:
        sys.path.insert(0, PKG_DIR)
    return importlib.import_module("packed")


@pytest.fixture(scope="module")
def rope_table(packed):
    return importlib.import_module("qk_prep").rope_table


@pytest.fixture(scope="module")
def capi():
    return importlib.import_module("610sample_b200.capi")


# ---- CPU ------------------------------------------------------------------------------------------

def _shape(capi, **over):
    s = capi.RopeShape()
    d = dict(n_tok=64, q_heads=4, k_heads=2, D=64, dtype=capi.ATTN_BF16, table_rows=64, axes=1, positions64=0, eps=1e-6)
    d.update({k: v for k, v in over.items() if k in d})
    for k, v in d.items():
        setattr(s, k, v)
    for i, v in enumerate(over.get("section", (d["D"] // 2,))):
        s.section[i] = v
    for i, h in enumerate((4, 2)):
        s.row_stride[i] = s.g_row_stride[i] = h * 64
        s.head_stride[i] = s.g_head_stride[i] = 64
    return s


@pytest.mark.parametrize("over, code, text", [
    (dict(dtype=9), -2, "dtype 9"), (dict(n_tok=-1), -1, "n_tok"), (dict(n_tok=2 ** 30 + 1), -1, "n_tok"), (dict(q_heads=-1), -1, "heads"),
    (dict(k_heads=2 ** 20 + 1), -1, "heads"), (dict(D=63), -1, "D must"), (dict(D=0), -1, "D must"), (dict(D=130), -1, "D must"),
    (dict(table_rows=-1), -1, "table_rows"), (dict(axes=0), -1, "axes"), (dict(axes=5), -1, "axes"), (dict(section=(31,)), -1, "sum to"),
    (dict(axes=2, section=(40, -8)), -1, "negative"), (dict(n_tok=2 ** 30, q_heads=2 ** 20), -5, "tiles"),
])
def test_refused_shapes(capi, over, code, text):
    L, one, s = capi.lib(), ctypes.c_void_p(4096), _shape(capi, **over)
    assert L.attn_b200_packed_qk_norm_rope(ctypes.byref(s), *([one] * 8), None) == code
    assert text in L.attn_b200_last_error().decode()
    assert L.attn_b200_packed_qk_norm_rope_backward(ctypes.byref(s), *([one] * 13), None) == code
    assert L.attn_b200_packed_qk_norm_rope_backward_scratch_bytes(ctypes.byref(s)) == 0


def test_refused_pointers(capi):
    L, good, odd = capi.lib(), ctypes.c_void_p(4096), ctypes.c_void_p(4097)
    s = _shape(capi)
    for i in range(8):
        for bad in (None, odd):
            if bad is None and i in (2, 3):
                continue      # no weight: no norm
            args = [good] * 8
            args[i] = bad
            assert L.attn_b200_packed_qk_norm_rope(ctypes.byref(s), *args, None) == -1
    args = [good] * 13
    args[2] = None
    assert L.attn_b200_packed_qk_norm_rope_backward(ctypes.byref(s), *args, None) == -1 and "not there" in L.attn_b200_last_error().decode()
    args = [good] * 12 + [None]
    assert L.attn_b200_packed_qk_norm_rope_backward(ctypes.byref(s), *args, None) == -1 and "scratch" in L.attn_b200_last_error().decode()
    assert L.attn_b200_packed_qk_norm_rope(ctypes.byref(_shape(capi, n_tok=0)), *([None] * 8), None) == 0
    assert L.attn_b200_packed_qk_norm_rope(ctypes.byref(_shape(capi, q_heads=0, k_heads=0)), *([None] * 8), None) == 0


def test_python_refusals(packed):
    x, f = torch.zeros(4, 2, 8), torch.zeros(4, 4, 2)
    with pytest.raises(ValueError, match="sections"):
        packed.packed_qk_norm_rope(x, x, None, None, f, torch.zeros(2, 4, dtype=torch.int32))
    with pytest.raises(RuntimeError, match="CUDA"):
        packed.packed_qk_norm_rope(x, x, None, None, f, torch.zeros(4, dtype=torch.int32))


# ---- against 64 bits ----------------------------------------------------------------------------------

def reference(x, w, g, table, positions, sections, eps):
    """(out, gx, gw) in 64 bits and bounds: f = 2^-24; a factor r of a sum of D squares is off by (D + 8) f, so a normed
    value by (D + 12) f, a turned pair by 2 f more of the sum of both products' sizes; then one rounding of the result.
    gx is a difference of two terms with such factors; gw a sum over all rows."""
    f, out_u = 2.0 ** -24, torch.finfo(x.dtype).eps / 2
    D = x.shape[2]
    x, g, table = x.double(), g.double(), table.double()
    pos = positions.reshape(-1, x.shape[0]).long()
    cs = torch.cat([t[p] for t, p in zip(table.split(list(sections), 1), pos)], 1)[:, None]
    c, s = cs[..., 0], cs[..., 1]
    turn = lambda a, b, c, s: torch.stack([a * c - b * s, a * s + b * c], -1).flatten(-2)
    size = lambda a, b: torch.stack([(a * c).abs() + (b * s).abs(), (a * s).abs() + (b * c).abs()], -1).flatten(-2)
    wd = w.double() if w is not None else None
    y = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + eps) * wd if w is not None else x
    a, b = y[..., 0::2], y[..., 1::2]
    out = turn(a, b, c, s)
    e_out = size(a, b) * (D + 16) * f + out_u * out.abs()
    ga, gb = g[..., 0::2], g[..., 1::2]
    gy, e_gy = turn(ga, gb, c, -s), size(ga, gb) * 4 * f
    if w is None:
        return (out, gy, None), (e_out, e_gy + out_u * gy.abs(), None)
    r = torch.rsqrt((x * x).mean(-1, keepdim=True) + eps)
    dot = (gy * wd * x).sum(-1, keepdim=True)
    sizes = ((gy.abs() * (D + 8) * f + e_gy) * (wd * x).abs()).sum(-1, keepdim=True)
    gx = r * gy * wd - x * r ** 3 / D * dot
    e_gx = r * (e_gy + gy.abs() * (D + 16) * f) * wd.abs() + x.abs() * r ** 3 / D * (sizes + dot.abs() * (3 * D + 40) * f) + out_u * gx.abs()
    rows = x.shape[0] * x.shape[1]
    gw = (gy * x * r).sum((0, 1))
    e_gw = ((e_gy + gy.abs() * (D + 16 + rows) * f) * (x * r).abs()).sum((0, 1)) + torch.finfo(w.dtype).eps / 2 * gw.abs()
    return (out, gx, gw), (e_out, e_gx, e_gw)


def inputs(n, H, Hkv, D, dtype, axes=1, seed=0, rows=500):
    gen = torch.Generator().manual_seed(seed)
    qkv = (torch.randn(n, H + 2 * Hkv, D, generator=gen) * 1.5).to(dtype).cuda()
    weights = [(1 + 0.2 * torch.randn(D, generator=gen)).to(dtype).cuda() for _ in range(2)]
    grads = [torch.randn(n, h, D, generator=gen).to(dtype).cuda() for h in (H, Hkv)]
    positions = torch.randint(0, rows, (axes, n) if axes > 1 else (n,), generator=gen, dtype=torch.int32).cuda()
    pairs = D // 2
    sections = {1: (pairs,), 2: (pairs // 3, pairs - pairs // 3), 3: (pairs // 4, pairs // 4, pairs - 2 * (pairs // 4)), 4: (0, 1, pairs - 2, 1)}[axes]
    return qkv[:, :H], qkv[:, H:H + Hkv], weights, grads, positions, sections


def both_passes(packed, q, k, weights, grads, table, positions, sections, eps=1e-6):
    leaves = [t.detach().requires_grad_(True) if t is not None else None for t in (q, k, *weights)]
    outs = packed.packed_qk_norm_rope(*leaves, table, positions, sections, eps)
    want = [t for t in leaves if t is not None]
    got = list(torch.autograd.grad(outs, want, grads))
    return [t.detach() for t in outs], [got.pop(0) if t is not None else None for t in leaves]


def check(packed, q, k, weights, grads, table, positions, sections, eps=1e-6):
    outs, gr = both_passes(packed, q, k, weights, grads, table, positions, sections, eps)
    plain = packed.packed_qk_norm_rope(q, k, *weights, table, positions, sections, eps)
    for i, x in enumerate((q, k)):
        want, bound = reference(x, weights[i], grads[i], table, positions, sections, eps)
        tiny = torch.finfo(x.dtype).smallest_normal * torch.finfo(x.dtype).eps
        assert torch.equal(plain[i], outs[i]) and outs[i].is_contiguous() and outs[i].shape == x.shape
        for name, a, b, e in zip(("out", "gx", "gw"), (outs[i], gr[i], gr[2 + i]), want, bound):
            assert (a is None) == (b is None)
            if a is not None and a.numel():
                assert a.dtype == (weights[i].dtype if name == "gw" else x.dtype)
                worst = ((a.double() - b).abs() / (e * 1.01 + tiny)).max()
                assert bool(worst <= 1), (i, name, float(worst))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("n, H, Hkv, D", [(1, 1, 1, 64), (33, 4, 2, 64), (65, 12, 12, 128), (130, 5, 1, 80), (31, 3, 2, 20), (40, 2, 2, 2),
                                          (17, 6, 3, 126), (700, 8, 8, 16), (9, 4, 0, 32), (9, 0, 3, 32)])
def test_sizes(packed, rope_table, dtype, n, H, Hkv, D):
    q, k, w, g, pos, sec = inputs(n, H, Hkv, D, dtype)
    check(packed, q, k, w, g, rope_table(D, 500, device="cuda"), pos, sec)


@pytest.mark.gpu
@pytest.mark.parametrize("axes, D", [(2, 64), (3, 128), (3, 80), (4, 64), (2, 30)])
@pytest.mark.parametrize("ptype", [torch.int32, torch.int64])
def test_axes(packed, rope_table, axes, D, ptype):
    q, k, w, g, pos, sec = inputs(77, 4, 2, D, torch.bfloat16, axes)
    check(packed, q, k, w, g, rope_table(D, 500, device="cuda"), pos.to(ptype), sec)


@pytest.mark.gpu
def test_weights(packed, rope_table):
    table = rope_table(64, 500, device="cuda")
    q, k, w, g, pos, sec = inputs(50, 4, 2, 64, torch.bfloat16)
    for ws in ((None, None), (w[0], None), (None, w[1]), (w[0].float(), w[1]), (w[0].float() + 1e-4, w[1].float())):
        check(packed, q, k, list(ws), g, table, pos, sec, eps=1e-3)
    q, k, w, g, pos, sec = inputs(50, 4, 2, 64, torch.float16)
    check(packed, q * 0 + q[:, :1] * 200, k * 1e-3, w, g, table, pos, sec, eps=0.0)


@pytest.mark.gpu
def test_strides(packed, rope_table):
    table = rope_table(64, 500, device="cuda")
    for dtype in (torch.bfloat16, torch.float32):
        q, k, w, g, pos, sec = inputs(45, 4, 2, 64, dtype)
        want = both_passes(packed, q.contiguous(), k.contiguous(), w, g, table, pos, sec)
        odd = torch.empty(45 * 4 * 65 + 1, device="cuda", dtype=dtype)[1:].view(45, 4, 65)[:, :, 1:]
        odd.copy_(q)
        first = torch.empty(2, 45, 64, device="cuda", dtype=dtype).transpose(0, 1)
        first.copy_(k)
        cols = torch.empty(45, 2, 128, device="cuda", dtype=dtype)[:, :, ::2]
        cols.copy_(k)
        gs = [torch.empty(45, h, 130, device="cuda", dtype=dtype)[:, :, 2:66].copy_(t) for h, t in zip((4, 2), g)]
        p2 = torch.stack([pos, pos], 1)[:, 0]
        for args in ((q, k, w, gs, table, pos, sec), (odd, first, w, g, table, p2, sec), (odd, cols, w, [g[0], g[1].transpose(0, 1).contiguous().transpose(0, 1)], table, pos, sec)):
            got = both_passes(packed, *args)
            for a, b in zip(got[0] + got[1][:2], want[0] + want[1][:2]):
                assert torch.equal(a, b)
            for a, b in zip(got[1][2:], want[1][2:]):
                assert torch.allclose(a, b, rtol=torch.finfo(dtype).eps * 2, atol=1e-4)      # the same sum


@pytest.mark.gpu
def test_positions_outside_of_the_table(packed, rope_table):
    q, k, w, g, pos, sec = inputs(20, 2, 1, 32, torch.bfloat16, rows=50)
    pos[3], pos[7], pos[9] = 50, -1, 2 ** 31 - 1
    a, b = packed.packed_qk_norm_rope(q, k, *w, rope_table(32, 50, device="cuda"), pos)
    for t in (a, b):
        assert t.isnan().flatten(1).any(1).nonzero().flatten().tolist() == [3, 7, 9]
    none = torch.zeros(0, 16, 2, device="cuda")
    assert bool(packed.packed_qk_norm_rope(q, k, *w, none, pos)[0].isnan().all())
    e = packed.packed_qk_norm_rope(q[:0], k[:0], *w, none, pos[:0])
    assert e[0].shape == (0, 2, 32)


@pytest.mark.gpu
def test_rows_without_gradient_have_no_influence(packed, rope_table):
    table = rope_table(64, 500, device="cuda")
    for dtype in (torch.bfloat16, torch.float32):
        q, k, w, g, pos, sec = inputs(90, 4, 2, 64, dtype)
        for t in g:
            t[60:] = 0
        want = both_passes(packed, q, k, w, g, table, pos, sec)[1]
        q[60:] = math.nan
        k[60:] = math.inf
        got = both_passes(packed, q, k, w, g, table, pos, sec)[1]
        for a, b in zip(got, want):
            assert torch.equal(a, b)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("D", [64, 128, 20])
@pytest.mark.parametrize("with_weights", [True, False])
def test_padding_behind_the_last_sequence_has_no_influence(packed, rope_table, dtype, D, with_weights):
    # rows that nothing reads: positions outside of the table, anything in q and k; first and second derivative
    table = rope_table(D, 500, device="cuda")
    q, k, w, g, pos, sec = inputs(90, 4, 2, D, dtype)
    u, v, uw, _, _, _ = inputs(90, 4, 2, D, dtype, seed=5)
    w = w if with_weights else [None, None]
    for t in (*g, u, v):
        t[60:] = 0

    def passes():
        leaves = [t.detach().clone().requires_grad_(True) for t in (q, k, *w) if t is not None]
        gl = [t.detach().clone().requires_grad_(True) for t in g]
        outs = packed.packed_qk_norm_rope(*leaves, *([None] * (4 - len(leaves))), table, pos, sec)
        plain = torch.autograd.grad(outs, leaves, gl, retain_graph=True)
        first = torch.autograd.grad(outs, leaves, gl, create_graph=True)
        second = torch.autograd.grad(first, leaves + gl, [u, v, *uw][:len(leaves)], allow_unused=True)
        return [*plain, *first, *[t for t in second if t is not None]]
    want = passes()
    pos[60:75], pos[75:] = -1, 2 ** 31 - 1
    q[60:70] = math.nan
    k[65:80] = math.inf
    got = passes()
    assert len(got) == len(want)
    for a, b in zip(got, want):
        assert bool(a.isfinite().all()) or a.shape[0] == 90
        assert torch.equal(a[:60], b[:60]) if a.shape[0] == 90 else torch.equal(a, b)
    for a in got[:2]:
        assert not bool(a[60:].any())


@pytest.mark.gpu
def test_refused_calls(packed, rope_table):
    q, k, w, g, pos, sec = inputs(20, 4, 2, 32, torch.bfloat16)
    t = rope_table(32, 500, device="cuda")
    f = packed.packed_qk_norm_rope
    for args, text in (((q, k[:10], *w, t, pos), "agree"), ((q, k.half(), *w, t, pos), "same dtype"), ((q, k, w[0][:8], w[1], t, pos), "weight must be"),
                       ((q, k, w[0].half(), w[1], t, pos), "weight must have"), ((q, k, *w, t[:, :8], pos), "freqs"), ((q, k, *w, t.half(), pos), "freqs"),
                       ((q, k, *w, t, pos.float()), "int32 or int64"), ((q, k, *w, t, pos[:5]), "n_tok"), ((q, k, *w, t, pos, (8, 8)), "sections"),
                       ((q, k, *w, t, pos, (15,)), "sum to"), ((q[0], k, *w, t, pos), "n_tok, heads"), ((q, k, *w, t, pos.cpu()), "CUDA")):
        with pytest.raises(RuntimeError, match=text):
            f(*args)
    with pytest.raises(RuntimeError, match="gradient of freqs"):
        f(q, k, *w, t.requires_grad_(True), pos)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype, tol", [(torch.float32, 1e-5), (torch.bfloat16, 1e-2)])
@pytest.mark.parametrize("with_weights", [True, False])
def test_second_derivative(packed, rope_table, dtype, tol, with_weights):
    q, k, w, g, pos, sec = inputs(40, 3, 2, 48, dtype, axes=3)
    w = w if with_weights else [None, None]
    u, v, uw, _, _, _ = inputs(40, 3, 2, 48, dtype, seed=4)
    table = rope_table(48, 500, device="cuda")
    leaves = [t.detach().clone().requires_grad_(True) for t in (q, k, *[x for x in w if x is not None])]
    gl = [t.requires_grad_(True) for t in g]
    args = leaves + [None] * (4 - len(leaves))
    first = torch.autograd.grad(packed.packed_qk_norm_rope(*args, table, pos, sec), leaves, gl, create_graph=True)
    tangents = [u, v, *uw][:len(leaves)]
    got = torch.autograd.grad(first, leaves + gl, tangents, allow_unused=True)
    d = [t.detach().double().requires_grad_(True) for t in leaves]
    gd = [t.detach().double().requires_grad_(True) for t in gl]
    cs = torch.cat([t[p.long()] for t, p in zip(table.double().split(list(sec), 1), pos)], 1)[:, None]

    def plain(x, wt):
        y = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-6) * wt if wt is not None else x
        a, b = y[..., 0::2], y[..., 1::2]
        return torch.stack([a * cs[..., 0] - b * cs[..., 1], a * cs[..., 1] + b * cs[..., 0]], -1).flatten(-2)
    dw = d[2:] if with_weights else [None, None]
    f64 = torch.autograd.grad([plain(d[0], dw[0]), plain(d[1], dw[1])], d, gd, create_graph=True)
    want = torch.autograd.grad(f64, d + gd, [t.double() for t in tangents], allow_unused=True)
    for a, b in zip(got, want):
        if b is None:
            assert a is None or not bool(a.any())
        else:
            assert float((a.double() - b).norm() / b.norm()) <= tol


@pytest.mark.gpu
def test_captured(packed, rope_table):
    table = rope_table(64, 500, device="cuda")
    q, k, w, g, pos, sec = inputs(300, 4, 2, 64, torch.bfloat16)
    flat = lambda r: r[0] + r[1]
    flat(both_passes(packed, q, k, w, g, table, pos, sec))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = flat(both_passes(packed, q, k, w, g, table, pos, sec))
    pos.copy_((pos * 7 + 3) % 500)
    for t in (q, k, *w, *g):
        t.copy_(torch.randn(t.shape))
    graph.replay()
    for a, b in zip(out, flat(both_passes(packed, q, k, w, g, table, pos, sec))):
        assert torch.equal(a, b)


# ---- the operators together -----------------------------------------------------------------------------

def layer_loss(ops, qkv_w, out_w, head, qw, kw, x, cu, targets, table, positions, H, Hkv):
    """One attention layer and the loss on a packed batch; ops: (norm + rotation, attention, loss)."""
    n, d = x.shape
    D = d // H
    qkv = torch.nn.functional.linear(x, qkv_w).view(n, H + 2 * Hkv, D)
    q, k = ops[0](qkv[:, :H], qkv[:, H:H + Hkv], qw, kw, table, positions)
    o = ops[1](q, k, qkv[:, H + Hkv:], cu)
    return ops[2](x + torch.nn.functional.linear(o.reshape(n, d), out_w), head, targets)


def plain_ops():
    def rope(q, k, qw, kw, table, positions):
        cs = table.to(q.dtype)[positions.long()][:, None]
        def one(x, w):
            y = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-6) * w
            a, b = y[..., 0::2], y[..., 1::2]
            return torch.stack([a * cs[..., 0] - b * cs[..., 1], a * cs[..., 1] + b * cs[..., 0]], -1).flatten(-2)
        return one(q, qw), one(k, kw)

    def attention(q, k, v, cu):
        out, cu = [], cu.tolist()
        for a, b in zip(cu[:-1], cu[1:]):
            kk, vv = (t[a:b].repeat_interleave(q.shape[1] // k.shape[1], 1).transpose(0, 1) for t in (k, v))
            S = q[a:b].transpose(0, 1) @ kk.transpose(1, 2) / math.sqrt(q.shape[2])
            S = S.masked_fill(torch.ones_like(S, dtype=torch.bool).triu(1), -math.inf)
            out.append((torch.softmax(S, -1) @ vv).transpose(0, 1))
        return torch.cat(out + [q.new_zeros(q.shape[0] - cu[-1], *q.shape[1:])])
    return rope, attention, lambda x, w, t: torch.nn.functional.cross_entropy(x @ w.T, t)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype, tol", [(torch.float32, 3e-5), (torch.bfloat16, 4e-2)])
def test_a_layer_and_its_loss(packed, rope_table, dtype, tol):
    # gradients, and gradients through one step of gradient descent, against the same layer in 64 bits, relative to the norm of each; bf16: some
    # ten roundings of 2^-8 behind one another on the way there and back
    lce = importlib.import_module("loss").linear_cross_entropy
    lens, H, Hkv, D, V = [70, 1, 130, 25], 4, 2, 32, 300
    cu = [0]
    for n in lens:
        cu.append(cu[-1] + n)
    n, d = cu[-1] + 6, H * D
    gen = torch.Generator().manual_seed(2)
    randn = lambda *shape, std=1.0: (torch.randn(*shape, generator=gen) * std).to(dtype).cuda()
    params = [randn((H + 2 * Hkv) * D, d, std=d ** -0.5), randn(d, d, std=d ** -0.5), randn(V, d, std=d ** -0.5), 1 + randn(D, std=0.1), 1 + randn(D, std=0.1)]
    x = randn(n, d)
    targets = torch.randint(0, V, (n,), generator=gen)
    positions = torch.cat([torch.arange(m) for m in lens] + [torch.zeros(6, dtype=torch.long)]).cuda()
    targets[[c - 1 for c in cu[1:]]] = -100
    targets[cu[-1]:] = -100
    targets = targets.cuda()
    table = rope_table(D, 200, device="cuda")
    cu_dev = torch.tensor(cu, dtype=torch.int32, device="cuda")
    plan = packed.packed_plan(cu_dev, n)
    own = (packed.packed_qk_norm_rope, lambda q, k, v, _: packed.packed_attention(q, k, v, plan), lce)

    def gradients(ops, params, x, table):
        params = [p.detach().requires_grad_(True) for p in params]
        loss = layer_loss(ops, *params[:3], *params[3:], x, cu_dev, targets, table, positions, H, Hkv)
        first = torch.autograd.grad(loss, params, create_graph=True)
        moved = [p - 0.3 * g for p, g in zip(params, first)]
        outer = layer_loss(ops, *moved[:3], *moved[3:], x, cu_dev, targets, table, positions, H, Hkv)
        return [loss.detach(), outer.detach(), *[t.detach() for t in first], *torch.autograd.grad(outer, params)]

    got = gradients(own, params, x, table)
    want = gradients(plain_ops(), [p.double() for p in params], x.double(), table.double())
    for a, b in zip(got, want):
        assert float((a.double() - b).norm() / b.norm()) <= tol
    # the rows of no sequence may hold anything
    x2 = x.clone()
    x2[cu[-1]:] = 1000.0
    again = gradients(own, params, x2, table)
    assert torch.equal(again[0], got[0])
