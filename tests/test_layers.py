"""Layer norm, linear layers and gated feed-forward blocks: refusals (CPU); results, both derivatives and differences against 64 bits with
bounds derived from the roundings; odd sizes, views, few rows, many tiles, streams, graphs, and the operators together (GPU)."""
import ctypes
import importlib
import math
import os
import sys

import pytest
import torch

PKG_DIR = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "610sample_b200")
HALF = [torch.bfloat16, torch.float16]
TYPES = HALF + [torch.float32]
ACTIVATIONS = [None, "silu", "gelu", "gelu_tanh"]


@pytest.fixture(scope="module")
def layers():
    if PKG_DIR not in sys.path:
        sys.path.insert(0, PKG_DIR)
    return importlib.import_module("layers")


@pytest.fixture(scope="module")
def capi():
    return importlib.import_module("610sample_b200.capi")


# ---- CPU ------------------------------------------------------------------------------------------

def _call(capi, dtype=None, form=0, kind=0, activation=0, count=1, rows=64, cols=128, k=96, pairs=1, ld=0, **over):
    c = capi.Products()
    c.dtype = capi.ATTN_BF16 if dtype is None else dtype
    c.form, c.kind, c.activation, c.count = form, kind, activation, count
    for i in range(min(max(count, 0), 3)):
        p = c.product[i]
        p.rows, p.cols, p.k, p.pairs = rows, cols, k, pairs
        for q in range(min(max(pairs, 0), 4)):
            p.pair[q] = capi.Factors(4096, 4096, ld or 128, ld or 128)
        p.out, p.ldo = 4096, ld or 128
    for name, value in over.items():
        setattr(c, name, value)
    return c


@pytest.mark.parametrize("over, code, text", [
    (dict(dtype=5), -2, "dtype 5"), (dict(form=3), -1, "form"), (dict(kind=3), -1, "kind"), (dict(activation=4), -1, "activation"),
    (dict(count=0), -1, "count"), (dict(count=4), -1, "count"), (dict(rows=-1), -1, "rows, cols and k"), (dict(cols=2 ** 30 + 1), -1, "rows, cols and k"),
    (dict(pairs=0), -1, "pairs"), (dict(pairs=5), -1, "pairs"), (dict(k=2 ** 29, pairs=4), -1, "k is too large"), (dict(count=3, pairs=3), -1, "pairs in all"),
    (dict(count=2, activation=1), -1, "several results"), (dict(count=2, bias=4096), -1, "several results"), (dict(kind=1, form=1), -1, "form NT"),
    (dict(kind=1, pairs=2), -1, "one pair"), (dict(kind=2), -1, "form NN"), (dict(kind=1, bias=4096), -1, "plain products"), (dict(k=0, activation=1), -1, "k must"),
    (dict(form=1, k=0, bias=4096), -1, "k must"),
])
def test_refused_products(capi, over, code, text):
    L, c = capi.lib(), _call(capi, **over)
    assert L.attn_b200_products(ctypes.byref(c), None, None) == code
    assert text in L.attn_b200_last_error().decode()
    assert L.attn_b200_products_scratch_bytes(ctypes.byref(c)) == 0


def test_refused_matrices(capi):
    L = capi.lib()

    def refused(c, text):
        assert L.attn_b200_products(ctypes.byref(c), None, None) == -1
        assert text in L.attn_b200_last_error().decode()

    for name in ("a", "b"):
        c = _call(capi)
        setattr(c.product[0].pair[0], name, None)
        refused(c, f"{name} is null")
        c = _call(capi)
        setattr(c.product[0].pair[0], name, 4104)
        refused(c, "16-byte")
        c = _call(capi, dtype=capi.ATTN_F32)
        setattr(c.product[0].pair[0], name, 4098)
        refused(c, "4-byte")
        c = _call(capi)
        setattr(c.product[0].pair[0], "ld" + name, 100)
        refused(c, "multiple of 8")
        c = _call(capi)
        setattr(c.product[0].pair[0], "ld" + name, 88)
        refused(c, "elements apart")
    c = _call(capi)
    c.product[0].out = None
    refused(c, "out is null")
    refused(_call(capi, residual=4096, ld_residual=64), "residual")
    refused(_call(capi, residual=4097, ld_residual=128), "residual")
    refused(_call(capi, kind=1, b2=None), "b2 is null")
    kept = (ctypes.c_void_p * 2)(4096, 4096)
    apart = (ctypes.c_int64 * 2)(128, 128)
    refused(_call(capi, kind=1, b2=4096, ldb2=128, kept=(ctypes.c_void_p * 2)(4096, None)), "together")
    refused(_call(capi, kind=1, b2=4096, ldb2=128, kept=kept, ld_kept=apart), "kept_low")
    refused(_call(capi, kind=1, b2=4096, ldb2=128, kept=kept, ld_kept=apart, kept_low=4096, ld_low=136), "kept_low")
    refused(_call(capi, kind=2, form=1, kept=kept, ld_kept=apart, kept_low=4096, ld_low=128), "out2 is null")
    refused(_call(capi, form=1, kept=kept, ld_kept=apart), "form NT only")
    # a long sum of few tiles is shared out, and needs scratch
    c = _call(capi, form=2, rows=256, cols=256, k=16384, ld=256)
    assert L.attn_b200_products_scratch_bytes(ctypes.byref(c)) > 0
    refused(c, "scratch")
    assert L.attn_b200_products(None, None, None) == -1


def test_refused_elements_and_norms(capi):
    L = capi.lib()

    def elements(text, code=-1, **over):
        e = capi.Elements()
        e.n, e.m, e.dtype, e.activation, e.pass_ = 8, 16, capi.ATTN_BF16, 1, 0
        for i in range(6):
            e.input[i], e.ld_input[i] = 4096, 16
        for i in range(5):
            e.out[i], e.ld_out[i] = 4096, 16
        for name, value in over.items():
            if name in ("input", "ld_input", "out"):
                getattr(e, name)[0] = value
            else:
                setattr(e, name, value)
        assert L.attn_b200_elements(ctypes.byref(e), None, None) == code
        assert text in L.attn_b200_last_error().decode()

    elements("dtype", -2, dtype=7)
    elements("pass", pass_=3)
    elements("activation", activation=9)
    elements("n and m", n=-1)
    elements("no sum", pass_=2, sum=4096)
    elements("null", input=None)
    elements("null", out=None)
    elements("elements apart", ld_input=8)
    elements("aligned", input=4097)
    elements("kept_low", pass_=2)
    assert L.attn_b200_elements(None, None, None) == -1
    for args, code in (((4096, 8, 4096, 16, 4, 9, 1), -1), ((4096, 16, 4096, 8, 4, 9, 1), -1), ((None, 16, 4096, 16, 4, 9, 1), -1), ((4097, 16, 4096, 16, 4, 9, 1), -1),
                       ((4096, 16, 4096, 16, -1, 9, 1), -1), ((4096, 16, 4096, 16, 4, 9, 7), -2)):
        assert L.attn_b200_copy_rows(*args, None) == code

    def shape(**over):
        d = dict(n=8, d=64, dtype=capi.ATTN_BF16, param_float=0, eps=1e-5, ld=64)
        d.update(over)
        return capi.NormShape(d["n"], d["d"], d["dtype"], d["param_float"], d["eps"], 0, d["ld"], d["ld"], d["ld"])

    one = ctypes.c_void_p(4096)
    for over, code, text in ((dict(dtype=4), -2, "dtype"), (dict(n=-1), -1, "n must"), (dict(d=0), -1, "d must"), (dict(d=32769), -1, "d must"),
                             (dict(ld=32), -1, "elements apart")):
        s = ctypes.byref(shape(**over))
        assert L.attn_b200_layer_norm(s, *([one] * 6), None) == code
        assert text in L.attn_b200_last_error().decode()
        assert L.attn_b200_layer_norm_backward(s, *([one] * 9), None) == code
        assert L.attn_b200_layer_norm_second_backward(s, *([one] * 12), None) == code
    s = ctypes.byref(shape())
    assert L.attn_b200_layer_norm(s, None, *([one] * 5), None) == -1
    assert L.attn_b200_layer_norm(s, *([one] * 5), None, None) == -1
    assert "together" in L.attn_b200_last_error().decode()
    assert L.attn_b200_layer_norm_backward(s, *([one] * 5), None, None, None, one, None) == -1
    assert "no gradient" in L.attn_b200_last_error().decode()
    assert L.attn_b200_layer_norm_backward(s, *([one] * 8), None, None) == -1
    assert "scratch" in L.attn_b200_last_error().decode()
    assert L.attn_b200_layer_norm_backward(s, *([one] * 3), None, *([one] * 5), None) == -1


def test_python_refusals(layers):
    x, w = torch.zeros(4, 8), torch.zeros(6, 8)
    with pytest.raises(ValueError, match="activation"):
        layers.linear(x, w, activation="tanh")
    with pytest.raises(ValueError, match="activation"):
        layers.gated_feed_forward(x, w, w, w.T, activation="relu6")
    for call in (lambda: layers.linear(x, w), lambda: layers.gated_feed_forward(x, w, w, w.T), lambda: layers.layer_norm(x)):
        with pytest.raises(RuntimeError, match="CUDA"):
            call()


# ---- against 64 bits ----------------------------------------------------------------------------------
# f = 2^-24; u: half a step of the type.  A sum of k products in fp32, in any order, is off by at most (k + 8) f of the sum of sizes (the tensor cores' by that
# and 2^-23 a block of 16 toward 0, which is within it).  The fast activations and their derivatives (ex2, rcp and the fitted polynomial) are within 1.2e-5 of the
# curve's own scale |z| (1 + |z|); the precise ones within 2^-20 of it.

F32 = 2.0 ** -24


def curve(z, kind):
    """(a, a', a'', bound of |a'|, of |a''|, of |a'''|) in 64 bits"""
    if kind is None:
        return z, torch.ones_like(z), torch.zeros_like(z)
    if kind == "gelu":
        F, d = 0.5 * torch.erfc(-z / math.sqrt(2)), torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
        return z * F, F + z * d, d * (2 - z * z)
    if kind == "silu":
        u, u1, u2 = z, torch.ones_like(z), torch.zeros_like(z)
    else:
        r = math.sqrt(8 / math.pi)
        u, u1, u2 = r * (z + 0.044715 * z ** 3), r * (1 + 3 * 0.044715 * z * z), r * 6 * 0.044715 * z
    s = torch.sigmoid(u)
    w = s * torch.sigmoid(-u)
    s1, s2 = w * u1, w * (1 - 2 * s) * u1 * u1 + w * u2
    return z * s, s + z * s1, 2 * s1 + z * s2


def curve_error(z, dtype):
    """What the kernels' activations and their derivatives may be off by, by itself."""
    return (1.2e-5 if dtype != torch.float32 else 2.0 ** -20) * torch.exp(-(z.abs() - 6).clamp(min=0)) * (1 + z.abs()) + 4 * F32 * z.abs()


def mm(a, ea, b, eb, k):
    """(a b, error): the factors are off by ea and eb, and the sum of k products by the rounding of fp32"""
    size = a.abs() @ b.abs()
    return a @ b, ea @ b.abs() + a.abs() @ eb + ea @ eb + (k + 8) * F32 * size


def rounded(v, e, dtype):
    """e of v once it has been rounded to the type"""
    info = torch.finfo(dtype)
    return e + (v.abs() + e) * info.eps / 2 + info.smallest_normal * info.eps


def near(got, want, error, what):
    assert got.shape == want.shape, what
    assert bool(got.isfinite().all()), what
    worst = ((got.double() - want).abs() / (error * 1.02 + 1e-30)).max() if want.numel() else torch.zeros(())
    assert bool(worst <= 1), (what, float(worst))


def inputs(shapes, dtype, seed=0):
    g = torch.Generator().manual_seed(seed)
    return [(torch.randn(*s, generator=g) * scale).to(dtype).cuda() for s, scale in shapes]


def linear_reference(x, w, b, r, g, kind, dtype):
    x, w, b, r, g = (t if t is None else t.double() for t in (x, w, b, r, g))
    zero = lambda t: torch.zeros_like(t)
    z, ez = mm(x, zero(x), w.T, zero(w.T), x.shape[1])
    if b is not None:
        z = z + b
        ez = ez + 2 * F32 * (z.abs() + b.abs())
    a, d1, d2 = curve(z, kind)
    own = curve_error(z, dtype) if kind else zero(z)
    ea = ez * 1.2 + own
    y = a if r is None else a + r
    ey = ea + 2 * F32 * y.abs()
    # z is kept in f16; |a''| <= 1.25 for all of them
    kept = ez if dtype == torch.float32 else rounded(z, ez, torch.float16)
    ed = own + (kept * 1.25 if kind else 0.0)
    dz = g * d1
    edz = rounded(dz, g.abs() * ed + 4 * F32 * dz.abs(), dtype) if kind else zero(dz)
    gx, egx = mm(dz, edz, w, zero(w), w.shape[0])
    gw, egw = mm(dz.T, edz.T, x, zero(x), x.shape[0])
    results = [(y, ey), (gx, egx), (gw, egw)]
    if b is not None:
        # summed before dz is rounded
        results.append((dz.sum(0), (g.abs() * ed + 4 * F32 * dz.abs()).sum(0) + (x.shape[0] + 8) * F32 * dz.abs().sum(0)))
    if r is not None:
        results.append((g, zero(g)))
    return [(v, rounded(v, e, dtype)) for v, e in results]


def passes(call, leaves, g):
    leaves = [t.detach().requires_grad_(True) for t in leaves]
    out = call(*leaves)
    return [out.detach(), *torch.autograd.grad(out, leaves, g)]


def check_linear(layers, n, k, m, dtype, kind, bias=True, residual=True, seed=0):
    x, w, b, r, g = inputs([((n, k), 1.0), ((m, k), 1.5 / math.sqrt(k)), ((m,), 0.5), ((n, m), 1.0), ((n, m), 1.0)], dtype, seed)
    b, r = b if bias else None, r if residual else None
    leaves = [t for t in (x, w, b, r) if t is not None]

    def call(x, w, *rest):
        rest = list(rest)
        bb = rest.pop(0) if bias else None
        return layers.linear(x, w, bb, kind, rest.pop(0) if residual else None)

    got = passes(call, leaves, g)
    want = linear_reference(x, w, b, r, g, kind, dtype)
    names = ["y", "gx", "gw"] + ["gb"] * bias + ["gr"] * residual
    for name, a, (v, e) in zip(names, got, want):
        assert a.dtype == dtype
        near(a, v, e, name)
    with torch.no_grad():
        assert torch.equal(call(*leaves), got[0])


SIZES = [(1, 1, 1), (1, 768, 264), (3, 8, 16), (8, 200, 33), (9, 72, 40), (16, 513, 300), (17, 96, 8), (32, 1100, 136), (33, 64, 256), (40, 7, 500), (127, 130, 65),
         (129, 72, 257), (256, 128, 256), (300, 777, 515), (513, 64, 1025)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n, k, m", SIZES)
def test_linear_sizes(layers, dtype, n, k, m):
    check_linear(layers, n, k, m, dtype, ACTIVATIONS[(n + m) % 4])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("kind", ACTIVATIONS)
@pytest.mark.parametrize("bias, residual", [(False, False), (True, False), (False, True)])
def test_linear_forms(layers, dtype, kind, bias, residual):
    for n in (5, 140):
        check_linear(layers, n, 136, 200, dtype, kind, bias, residual, seed=n)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("n, k, m", [(5000, 768, 520), (200, 3000, 768), (9000, 264, 264), (300, 2048, 20000), (2100, 64, 10000), (20, 9000, 700), (6, 300, 12000), (20, 4000, 9600)])
def test_linear_many_tiles_and_shares(layers, dtype, n, k, m):
    # several rounds of tiles, sums shared out along k with an epilogue behind them, few rows against long and against wide weights
    check_linear(layers, n, k, m, dtype, "gelu")


def gated_reference(x, wg, wu, wd, r, g, kind, dtype):
    x, wg, wu, wd, r, g = (t if t is None else t.double() for t in (x, wg, wu, wd, r, g))
    zero = lambda t: torch.zeros_like(t)
    z, ez = mm(x, zero(x), wg.T, zero(wg.T), x.shape[1])
    u, eu = mm(x, zero(x), wu.T, zero(wu.T), x.shape[1])
    a, d1, _ = curve(z, kind)
    own = curve_error(z, dtype)
    ea = ez * 1.2 + own
    h = a * u
    eh = rounded(h, ea * (u.abs() + eu) + a.abs() * eu + 4 * F32 * h.abs(), dtype)
    y, ey = mm(h, eh, wd.T, zero(wd.T), wd.shape[1])
    if r is not None:
        y = y + r
        ey = ey + 2 * F32 * (y.abs() + r.abs())
    # z and u are kept with 11 bits of mantissa (bf16; cut off, and read as the middle), 14 (f16)
    step = {torch.bfloat16: 2.0 ** -12, torch.float16: 2.0 ** -15, torch.float32: 0.0}[dtype]
    tiny = 2.0 ** -28 if dtype == torch.float16 else 0.0
    kz, ku = ez + step * (z.abs() + ez) + tiny, eu + step * (u.abs() + eu) + tiny
    ea, ed = kz * 1.2 + own, kz * 1.25 + own
    gh, egh = mm(g, zero(g), wd, zero(wd), wd.shape[0])
    dz, du = gh * d1 * u, gh * a
    edz = rounded(dz, egh * (d1 * u).abs() + (gh.abs() + egh) * (ed * (u.abs() + ku) + d1.abs() * ku) + 6 * F32 * dz.abs(), dtype)
    edu = rounded(du, egh * a.abs() + (gh.abs() + egh) * ea + 4 * F32 * du.abs(), dtype)
    gx1, e1 = mm(dz, edz, wg, zero(wg), 2 * wg.shape[0])
    gx2, e2 = mm(du, edu, wu, zero(wu), 2 * wg.shape[0])
    results = [(y, ey), (gx1 + gx2, e1 + e2), mm(dz.T, edz.T, x, zero(x), x.shape[0]), mm(du.T, edu.T, x, zero(x), x.shape[0]), mm(g.T, zero(g.T), h, eh, x.shape[0])]
    if r is not None:
        results.append((g, zero(g)))
    return [(v, rounded(v, e, dtype)) for v, e in results]


def gated_inputs(n, d, f, m, dtype, seed=0):
    return inputs([((n, d), 1.0), ((f, d), 1.5 / math.sqrt(d)), ((f, d), 1.5 / math.sqrt(d)), ((m, f), 1 / math.sqrt(f)), ((n, m), 1.0), ((n, m), 1.0)], dtype, seed)


def check_gated(layers, n, d, f, m, dtype, kind, residual=True):
    x, wg, wu, wd, r, g = gated_inputs(n, d, f, m, dtype)
    leaves = [x, wg, wu, wd] + [r] * residual
    call = lambda x, a, b, c, r=None: layers.gated_feed_forward(x, a, b, c, kind, r)
    got = passes(call, leaves, g)
    for name, a, (v, e) in zip(("y", "gx", "gg", "gu", "gd", "gr"), got, gated_reference(x, wg, wu, wd, r if residual else None, g, kind, dtype)):
        assert a.dtype == dtype
        near(a, v, e, name)
    with torch.no_grad():
        assert torch.equal(call(*leaves), got[0])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n, d, f, m", [(1, 1, 1, 1), (1, 256, 300, 256), (7, 40, 72, 24), (16, 100, 33, 7), (30, 136, 344, 136), (33, 72, 200, 80), (128, 64, 128, 64), (129, 65, 130, 61),
                                        (260, 264, 500, 264), (600, 96, 1032, 96)])
def test_gated_sizes(layers, dtype, n, d, f, m):
    check_gated(layers, n, d, f, m, dtype, ACTIVATIONS[1 + (n + f) % 3], residual=n % 2 == 0)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("kind", ACTIVATIONS)
def test_gated_activations(layers, dtype, kind):
    check_gated(layers, 150, 72, 264, 72, dtype, kind)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("n, d, f", [(3000, 264, 2048), (20, 2000, 5000), (2500, 768, 768)])
def test_gated_many_tiles(layers, dtype, n, d, f):
    check_gated(layers, n, d, f, d, dtype, "silu")


def norm_reference(x, w, b, g, eps, dtype, ptype):
    x, w, b, g = (t if t is None else t.double() for t in (x, w, b, g))
    n, d = x.shape
    mean = x.mean(1, keepdim=True)
    size = x.abs().amax(1, keepdim=True)
    c = x - mean
    var = (c * c).mean(1, keepdim=True)
    r = (var + eps).rsqrt()
    xh = c * r
    # the mean is off by (d + 2) f of the sizes' mean at most, and x - mean is rounded; r relatively by half of what the variance is, and a few f
    em = (d + 2) * F32 * x.abs().mean(1, keepdim=True) + 2 * F32 * size
    er = (2 * em * c.abs().mean(1, keepdim=True) + em * em + (d + 4) * F32 * var) / (2 * (var + eps)) + 6 * F32
    exh = em * r + xh.abs() * er + 4 * F32 * xh.abs()
    ones = torch.ones(d, dtype=torch.float64, device="cuda")
    ww, bb = ones if w is None else w, 0 * ones if b is None else b
    y = xh * ww + bb
    results = [(y, exh * ww.abs() + 4 * F32 * (y.abs() + bb.abs()))]
    cg = g * ww
    m0, m1 = cg.mean(1, keepdim=True), (cg * xh).mean(1, keepdim=True)
    e0 = (d + 4) * F32 * cg.abs().mean(1, keepdim=True)
    e1 = (cg.abs() * exh).mean(1, keepdim=True) + (d + 6) * F32 * (cg * xh).abs().mean(1, keepdim=True)
    gx = r * (cg - m0 - xh * m1)
    egx = r * (1 + er) * (e0 + exh * (m1.abs() + e1) + xh.abs() * e1 + 6 * F32 * (cg.abs() + m0.abs() + (xh * m1).abs())) + gx.abs() * er
    results.append((gx, egx))
    if w is not None:
        results.append(((g * xh).sum(0), (g.abs() * exh).sum(0) + (n + 8) * F32 * (g * xh).abs().sum(0)))
    if b is not None:
        results.append((g.sum(0), (n + 8) * F32 * g.abs().sum(0)))
    return [(v, rounded(v, e, t)) for (v, e), t in zip(results, (dtype, dtype, ptype, ptype))]


def norm_inputs(n, d, dtype, ptype, seed=0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(n, d, generator=g) * (torch.rand(n, 1, generator=g) * 3 + 0.3) + torch.randn(n, 1, generator=g) * 2
    w, b = torch.randn(d, generator=g) * 0.3 + 1, torch.randn(d, generator=g) * 0.3
    return x.to(dtype).cuda(), w.to(ptype).cuda(), b.to(ptype).cuda(), torch.randn(n, d, generator=g).to(dtype).cuda()


def check_norm(layers, n, d, dtype, ptype=None, weight=True, bias=True, eps=1e-5):
    ptype = ptype or dtype
    x, w, b, g = norm_inputs(n, d, dtype, ptype)
    w, b = w if weight else None, b if bias else None

    def call(x, *rest):
        rest = list(rest)
        ww = rest.pop(0) if weight else None
        return layers.layer_norm(x, ww, rest.pop(0) if bias else None, eps)

    leaves = [t for t in (x, w, b) if t is not None]
    got = passes(call, leaves, g)
    for name, a, (v, e) in zip(["y", "gx"] + ["gw"] * weight + ["gb"] * bias, got, norm_reference(x, w, b, g, eps, dtype, ptype)):
        assert a.dtype == (dtype if name in ("y", "gx") else ptype)
        near(a, v, e, name)
    with torch.no_grad():
        assert torch.equal(call(*leaves), got[0])


NORM_WIDTHS = [1, 2, 7, 8, 100, 256, 257, 512, 520, 768, 777, 1024, 1030, 2048, 2056, 4096, 5000, 8192, 8200, 16384, 16392, 32768]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d", NORM_WIDTHS)
def test_norm_widths(layers, dtype, d):
    check_norm(layers, 37 if d < 5000 else 5, d, dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n", [1, 2, 9, 600, 2500])
def test_norm_rows(layers, dtype, n):
    for d in (64, 768, 1024):
        check_norm(layers, n, d, dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d", [99, 768])
def test_norm_parameters(layers, dtype, d):
    for weight, bias in ((False, False), (True, False), (False, True)):
        check_norm(layers, 50, d, dtype, None, weight, bias, eps=1e-3)
    check_norm(layers, 50, d, dtype, torch.float32)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_norm_of_equal_values(layers, dtype):
    # no variance: the centred row is 0, and r = 1 / sqrt(eps)
    x = torch.full((5, 96), 3.0, device="cuda", dtype=dtype)
    w, b = torch.full((96,), 2.0, device="cuda", dtype=dtype), torch.full((96,), 0.5, device="cuda", dtype=dtype)
    out, gx, gw, gb = passes(lambda x, w, b: layers.layer_norm(x, w, b), [x, w, b], torch.ones_like(x))
    assert bool((out == 0.5).all()) and not bool(gx.any()) and not bool(gw.any()) and bool((gb == 5).all())


# ---- second derivatives -----------------------------------------------------------------------------------

def second(call, leaves, g, tangents, define):
    """(derivative of <first gradients, tangents> in the leaves and g, the same in 64 bits)"""
    a = [t.detach().requires_grad_(True) for t in leaves + [g]]
    first = torch.autograd.grad(call(*a[:-1]), a[:-1], a[-1], create_graph=True)
    want_of = [t.detach().double().requires_grad_(True) for t in leaves + [g]]
    f64 = torch.autograd.grad(define(*want_of[:-1]), want_of[:-1], want_of[-1], create_graph=True)
    pick = [i for i, t in enumerate(tangents) if t is not None]
    got = torch.autograd.grad([first[i] for i in pick], a, [tangents[i] for i in pick], allow_unused=True)
    want = torch.autograd.grad([f64[i] for i in pick], want_of, [tangents[i].double() for i in pick], allow_unused=True)
    return got, want


# a gradient is the sum of up to three terms of factors that have been rounded four times at most, each by half a step; the terms may cancel to a third of their size
SECOND = {torch.bfloat16: 4 * 3 * 2.0 ** -8 / math.sqrt(3), torch.float16: 4 * 3 * 2.0 ** -11 / math.sqrt(3), torch.float32: 3e-5}


def close(got, want, dtype, least=0.0):
    for i, (a, b) in enumerate(zip(got, want)):
        if b is None or a is None:
            assert (a is None or not bool(a.any())) and (b is None or not bool(b.any())), i
            continue
        assert a.shape == b.shape and bool(a.isfinite().all())
        assert float((a.double() - b).norm()) <= max(SECOND[dtype], least) * float(b.norm()) + 1e-12, (i, float((a.double() - b).norm() / b.norm()))


def define_act(z, kind):
    return {None: lambda z: z, "silu": torch.nn.functional.silu, "gelu": torch.nn.functional.gelu,
            "gelu_tanh": lambda z: torch.nn.functional.gelu(z, approximate="tanh")}[kind](z)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("kind", ACTIVATIONS)
@pytest.mark.parametrize("n, k, m", [(60, 48, 90), (5, 33, 41), (300, 264, 136)])
def test_linear_second_derivative(layers, dtype, kind, n, k, m):
    leaves = inputs([((n, k), 1.0), ((m, k), 1.5 / math.sqrt(k)), ((m,), 0.5), ((n, m), 1.0)], dtype)
    g, = inputs([((n, m), 1.0)], dtype, 5)
    tangents = inputs([((n, k), 1.0), ((m, k), 1.0), ((m,), 1.0), ((n, m), 1.0)], dtype, 6)
    call, define = lambda x, w, b, r: layers.linear(x, w, b, kind, r), lambda x, w, b, r: define_act(x @ w.T + b, kind) + r
    close(*second(call, leaves, g, tangents, define), dtype)
    for alone in range(3):      # a cotangent of one gradient only
        close(*second(call, leaves, g, [t if i == alone else None for i, t in enumerate(tangents)], define), dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("kind", ACTIVATIONS)
@pytest.mark.parametrize("n, d, f", [(40, 48, 72), (5, 33, 41), (200, 136, 264)])
def test_gated_second_derivative(layers, dtype, kind, n, d, f):
    x, wg, wu, wd, r, g = gated_inputs(n, d, f, d, dtype)
    tangents = gated_inputs(n, d, f, d, dtype, 9)[:5]
    call = lambda x, a, b, c, r: layers.gated_feed_forward(x, a, b, c, kind, r)
    define = lambda x, a, b, c, r: (define_act(x @ a.T, kind) * (x @ b.T)) @ c.T + r
    close(*second(call, [x, wg, wu, wd, r], g, tangents, define), dtype)
    for alone in range(4):
        close(*second(call, [x, wg, wu, wd, r], g, [t if i == alone else None for i, t in enumerate(tangents)], define), dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n, d", [(40, 768), (70, 99), (3, 8192), (600, 256), (4, 20000)])
def test_norm_second_derivative(layers, dtype, n, d):
    # every term has a mean over the row of products that are independent of each other, of sizes s on average: the mean is about s / sqrt(d), its rounding
    # up to (32 + 10) f s, with 32 elements to a thread and ten steps between threads.  So relatively 42 f sqrt(d)
    sums = 42 * F32 * math.sqrt(d)
    x, w, b, g = norm_inputs(n, d, dtype, dtype)
    tangents = norm_inputs(n, d, dtype, dtype, 7)[:3]
    call, define = lambda x, w, b: layers.layer_norm(x, w, b), lambda x, w, b: torch.nn.functional.layer_norm(x, (d,), w, b)
    close(*second(call, [x, w, b], g, tangents, define), dtype, sums)
    for alone in range(3):
        close(*second(call, [x, w, b], g, [t if i == alone else None for i, t in enumerate(tangents)], define), dtype, sums)
    x, _, _, g = norm_inputs(n, d, dtype, dtype, 3)
    close(*second(lambda x: layers.layer_norm(x), [x], g, [tangents[0]], lambda x: torch.nn.functional.layer_norm(x, (d,))), dtype, sums)


@pytest.mark.gpu
def test_no_third_derivative(layers):
    x, w, g = inputs([((6, 16), 1.0), ((8, 16), 1.0), ((6, 8), 1.0)], torch.float32)
    wd, = inputs([((8, 8), 1.0)], torch.float32, 1)
    for call, leaves in ((lambda x, w: layers.linear(x, w, activation="silu"), [x, w]), (lambda x, w: layers.layer_norm(layers.linear(x, w)), [x, w]),
                         (lambda x, w, v: layers.gated_feed_forward(x, w, w, v), [x, w, wd])):
        leaves = [t.detach().requires_grad_(True) for t in leaves]
        first = torch.autograd.grad(call(*leaves), leaves, g, create_graph=True)
        with pytest.raises(RuntimeError, match="third derivative"):
            torch.autograd.grad(sum((t * t).sum() for t in first), leaves, create_graph=True)


@pytest.mark.gpu
def test_gradients_against_differences(layers):
    # h = 2^-6: the truncation is h^2 / 6 of a third derivative of the order of the first; rounding of the sum of n m results, relatively 2^-24 sqrt(n m), over 2 h
    h = 2.0 ** -6
    x, w, b, g = inputs([((40, 24), 1.0), ((32, 24), 0.3), ((32,), 0.5), ((40, 32), 1.0)], torch.float32)
    wd, nw, nb = inputs([((24, 32), 0.2), ((24,), 0.3), ((24,), 0.3)], torch.float32, 2)
    gd, = inputs([((40, 24), 1.0)], torch.float32, 3)
    for call, leaves, up in ((lambda x, w, b: layers.linear(x, w, b, "gelu"), [x, w, b], g), (lambda x, w, v: layers.gated_feed_forward(x, w, w.flip(0), v), [x, w, wd], gd),
                             (lambda x, a, c: layers.layer_norm(x, a, c), [x, nw, nb], gd)):
        grads = passes(call, leaves, up)[1:]
        for i, (t, grad) in enumerate(zip(leaves, grads)):
            move, = inputs([(tuple(t.shape), 1.0)], torch.float32, 11 + i)
            at = lambda s: (call(*[v + s * move if j == i else v for j, v in enumerate(leaves)]).double() * up.double()).sum()
            want = float((at(h) - at(-h)) / (2 * h))
            got = float((grad.double() * move.double()).sum())
            assert abs(got - want) <= 5e-3 * float(grad.double().norm() * move.double().norm()), (i, got, want)


# ---- how they are called ------------------------------------------------------------------------------------

def whole(layers, dtype, n=200, d=136, f=264, seed=0):
    """Inputs, and a layer's steps with all gradients, of one type."""
    x, wg, wu, wd, r, g = gated_inputs(n, d, f, d, dtype, seed)
    w1, b1 = inputs([((f, d), 1 / math.sqrt(d)), ((f,), 0.3)], dtype, seed + 50)
    w2, nw, nb = inputs([((d, f), 1 / math.sqrt(f)), ((d,), 0.3), ((d,), 0.3)], dtype, seed + 51)
    tensors = [x, wg, wu, wd, w1, b1, w2, nw, nb]

    def step():
        t = [v.detach().requires_grad_(True) for v in tensors]
        x, wg, wu, wd, w1, b1, w2, nw, nb = t
        y = layers.linear(layers.linear(layers.layer_norm(x, nw, nb), w1, b1, "gelu"), w2, residual=x)
        y = layers.gated_feed_forward(layers.layer_norm(y, nw), wg, wu, wd, residual=y)
        return [y.detach(), *torch.autograd.grad(y, t, g)]

    return tensors + [g], step


@pytest.mark.gpu
@pytest.mark.parametrize("dtype, tol", [(torch.float32, 2e-5), (torch.bfloat16, 4e-2), (torch.float16, 5e-3)])
def test_a_layer(layers, dtype, tol):
    # against the same in 64 bits: about ten roundings of half a step one behind the other, and gradients that meet
    tensors, step = whole(layers, dtype)
    got = step()
    t = [v.double().requires_grad_(True) for v in tensors[:-1]]
    x, wg, wu, wd, w1, b1, w2, nw, nb = t
    F = torch.nn.functional
    y = F.gelu(F.layer_norm(x, (136,), nw, nb) @ w1.T + b1) @ w2.T + x
    h = F.layer_norm(y, (136,), nw)
    y = (F.silu(h @ wg.T) * (h @ wu.T)) @ wd.T + y
    for a, b in zip(got, [y.detach(), *torch.autograd.grad(y, t, tensors[-1].double())]):
        assert float((a.double() - b).norm() / b.norm()) <= tol


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n", [3, 200])
def test_captured_and_on_two_streams(layers, dtype, n):
    tensors, step = whole(layers, dtype, n)
    step()
    torch.cuda.synchronize()
    graphs = [torch.cuda.CUDAGraph() for _ in range(2)]      # two graphs of the same leaves
    outs = []
    for graph in graphs:
        with torch.cuda.graph(graph):
            outs.append(step())
    for seed in (1, 2):
        fresh, _ = whole(layers, dtype, n, seed=seed)
        for t, s in zip(tensors, fresh):
            t.copy_(s)
        for graph in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for a, b, c in zip(*outs, step()):
            assert torch.equal(a, c) and torch.equal(b, c)
    cases = [whole(layers, dtype, n + 60 * i, seed=7 + i)[1] for i in range(2)]
    want = [c() for c in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    for _ in range(4):
        got = []
        for st, c in zip(streams, cases):
            with torch.cuda.stream(st):
                got.append(c())
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert all(torch.equal(p, q) for p, q in zip(a, b))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n", [6, 90])
def test_views(layers, dtype, n):
    x, wg, wu, wd, r, g = gated_inputs(n, 64, 96, 64, dtype)
    w, b = inputs([((96, 64), 0.2), ((96,), 0.3)], dtype, 4)
    res, gf = inputs([((n, 96), 1.0), ((n, 96), 1.0)], dtype, 5)
    nw = b[:64].contiguous()

    def same(got, want):
        # products: the same bits.  The norm (the last three) takes rows that no 16-byte load reads element by element, in another order: every sum of 64 values and
        # what follows from it, of at most eight times the largest result, is off by that many roundings in either, and the results may be rounded to either side
        for i, (p, q) in enumerate(zip(got, want)):
            p = p.reshape(q.shape)
            if i < len(want) - 3:
                assert torch.equal(p, q), i
            else:
                assert bool(((p.double() - q.double()).abs() <= torch.finfo(dtype).eps * q.double().abs() + 2 * 72 * F32 * 8 * q.double().abs().max()).all()), i

    def run(x, w, b, res, wg, wu, wd, r, nw, gf, g):
        return passes(lambda x, w, b, r: layers.linear(x, w, b, "gelu", r), [x, w, b, res], gf) + passes(
            lambda *t: layers.gated_feed_forward(*t[:4], residual=t[4]), [x, wg, wu, wd, r], g) + passes(lambda x, w: layers.layer_norm(x, w), [x, nw], g)

    plain = run(x, w, b, res, wg, wu, wd, r, nw, gf, g)

    def inside(t, extra, offset):      # a slice of wider rows, from an odd element or one that 16 bytes divide
        wide = torch.full((t.shape[0], t.shape[1] + extra), float("nan"), device="cuda", dtype=t.dtype)
        view = wide[:, offset:offset + t.shape[1]]
        view.copy_(t)
        return view

    for extra, offset in ((8, 0), (16, 8), (5, 1), (3, 3)):
        t = [v if v.dim() == 1 else inside(v, extra, offset) for v in (x, w, b, res, wg, wu, wd, r, nw, gf, g)]
        t[2] = torch.stack([b, b], 1)[:, 0]
        same(run(*t), plain)
    same(run(x, w.T.contiguous().T, b, res, wg.T.contiguous().T, wu, wd.T.contiguous().T, r.T.contiguous().T, nw, gf, g.T.contiguous().T), plain)
    # leading axes, and an expanded gradient
    shape = lambda t: t.view(2, n // 2, t.shape[1]) if t.dim() == 2 and t.shape[0] == n else t
    same(run(*[shape(v) for v in (x, w, b, res, wg, wu, wd, r, nw, gf, g)]), plain)
    one = passes(lambda x, w: layers.linear(x, w), [x, w], torch.ones(n, 96, device="cuda", dtype=dtype))
    leaves = [t.detach().requires_grad_(True) for t in (x, w)]
    for p, q in zip(torch.autograd.grad(layers.linear(*leaves).sum(), leaves), one[1:]):
        assert torch.equal(p, q)
    assert layers.linear(x[0], w, b).shape == (96,) and layers.layer_norm(x[0]).shape == (64,)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_no_rows(layers, dtype):
    x, wg, wu, wd, r, g = gated_inputs(0, 16, 24, 16, dtype)
    b, = inputs([((24,), 1.0)], dtype)
    for call, leaves, up in ((lambda x, w, b: layers.linear(x, w, b, "silu"), [x, wg, b], torch.zeros(0, 24, device="cuda", dtype=dtype)),
                             (lambda x, w: layers.linear(x, w), [x, wg], torch.zeros(0, 24, device="cuda", dtype=dtype)),
                             (lambda *t: layers.gated_feed_forward(*t), [x, wg, wu, wd], g), (lambda x, w, b: layers.layer_norm(x, w, b), [x, b[:16], b[8:]], g)):
        out, *grads = passes(call, leaves, up)
        assert out.shape[0] == 0
        for t, grad in zip(leaves, grads):
            assert grad.shape == t.shape and not bool(grad.any())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_some_gradients_only(layers, dtype):
    x, wg, wu, wd, r, g = gated_inputs(140, 64, 96, 64, dtype)
    b, = inputs([((96,), 0.3)], dtype)
    gf, = inputs([((140, 96), 1.0)], dtype, 3)
    for call, tensors, up in ((lambda x, w, b: layers.linear(x, w, b, "gelu"), [x, wg, b], gf), (lambda x, w, b: layers.linear(x, w, b), [x, wg, b], gf),
                              (lambda *t: layers.gated_feed_forward(*t[:4], residual=t[4]), [x, wg, wu, wd, r], g),
                              (lambda x, w, b: layers.layer_norm(x, w, b), [x, b[:64], b[32:]], g), (lambda x, b: layers.layer_norm(x, None, b), [x, b[:64]], g)):
        every = passes(call, tensors, up)[1:]
        for i, want in enumerate(every):
            t = [v.detach().requires_grad_(j == i) for j, v in enumerate(tensors)]
            got, = torch.autograd.grad(call(*t), t[i], up)
            assert torch.equal(got, want), i


@pytest.mark.gpu
def test_results_leave_what_lies_between_their_rows(layers, capi):
    # through the C ABI: a result that is a slice of wider rows, and a row behind its last one.  Written up to a multiple of 8 columns
    n, k, m = 130, 72, 100
    x, w = inputs([((n, k), 1.0), ((m, k), 0.2)], torch.bfloat16)
    wt = torch.nn.functional.pad(w.T, (0, 4)).contiguous()      # [k, m] in rows of 104
    for form, a, b, rows, cols, kk, product in ((0, x, w, n, m, k, lambda p, q: p @ q.T), (1, x, wt, n, m, k, lambda p, q: p @ q[:, :m]), (2, x, x, k, k, n, lambda p, q: p.T @ q)):
        wide = torch.full((rows + 1, 120), 7.0, device="cuda", dtype=torch.bfloat16)
        c = _call(capi, form=form, rows=rows, cols=cols, k=kk)
        c.product[0].pair[0] = capi.Factors(a.data_ptr(), b.data_ptr(), a.stride(0), b.stride(0))
        c.product[0].out, c.product[0].ldo = wide.data_ptr(), 120
        scratch = torch.empty(capi.lib().attn_b200_products_scratch_bytes(ctypes.byref(c)) + 16, dtype=torch.uint8, device="cuda")
        capi.check(capi.lib().attn_b200_products(ctypes.byref(c), scratch.data_ptr(), torch.cuda.current_stream().cuda_stream), "products")
        want, size = product(a.double(), b.double()), product(a.double().abs(), b.double().abs())
        near(wide[:rows, :cols], want, rounded(want, (kk + 8) * F32 * size, torch.bfloat16), form)
        assert bool((wide[:rows, (cols + 7) // 8 * 8:] == 7).all()) and bool((wide[rows] == 7).all())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n", [5, 20, 150])
def test_what_lies_behind_odd_rows_has_no_influence(layers, dtype, n):
    # widths that are no multiple of 8, read in place from rows that go on with NaN
    def rows(t):
        wide = torch.full((t.shape[0], (t.shape[1] + 7) // 8 * 8), float("nan"), device="cuda", dtype=dtype)
        wide[:, :t.shape[1]] = t
        return wide[:, :t.shape[1]]

    x, wg, wu, wd, r, g = gated_inputs(n, 100, 133, 99, dtype)
    call = lambda *t: layers.gated_feed_forward(*t[:4], residual=t[4])
    for a, b in zip(passes(call, [x, wg, wu, wd, r], g), passes(call, [rows(t) for t in (x, wg, wu, wd, r)], rows(g))):
        assert torch.equal(a, b)
    call = lambda x, w, r: layers.linear(x, w, None, "silu", r)
    w, = inputs([((99, 100), 0.2)], dtype, 3)
    for a, b in zip(passes(call, [x, w, r], g), passes(call, [rows(t) for t in (x, w, r)], rows(g))):
        assert torch.equal(a, b)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_rows_do_not_reach_each_other(layers, dtype):
    # infinities and NaN in some rows stay there: results and the gradients of the rows themselves
    x, wg, wu, wd, r, g = gated_inputs(200, 64, 96, 64, dtype)
    bad = torch.zeros(200, dtype=torch.bool, device="cuda")
    bad[[0, 31, 128, 199]] = True
    dirty = torch.where(bad[:, None], torch.tensor(float("nan"), device="cuda", dtype=dtype), x)
    dirty[31] = float("inf")
    for call in (lambda t: layers.linear(t, wg, activation="gelu"), lambda t: layers.gated_feed_forward(t, wg, wu, wd), lambda t: layers.layer_norm(t)):
        up = torch.ones_like(call(x))
        clean, soiled = passes(call, [x], up), passes(call, [dirty], up)
        for a, b in zip(clean, soiled):
            assert torch.equal(a[~bad], b[~bad])
        assert not bool(soiled[0][bad].isfinite().all())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("kind", ["silu", "gelu", "gelu_tanh"])
def test_large_arguments(layers, dtype, kind):
    # one input times one weight: z over the type's range, and the curve's ends: z or 0, slope 1 or 0
    top = min(torch.finfo(dtype).max / 2, 1e30)
    z = torch.cat([-torch.logspace(-4, math.log10(top), 200), torch.zeros(1), torch.logspace(-4, math.log10(top), 200)]).to(dtype).cuda()
    for n in (401, 5):      # in tiles, and few rows
        x, w = z[:n, None].contiguous() if n > 32 else torch.ones(n, 1, device="cuda", dtype=dtype), torch.ones(8, 1, device="cuda", dtype=dtype) if n > 32 else z[:, None].contiguous()
        zz = x.double() @ w.double().T
        y, gx, gw = passes(lambda x, w: layers.linear(x, w, activation=kind), [x, w], torch.ones(n, w.shape[0], device="cuda", dtype=dtype) / 8)
        a, d1, _ = curve(zz, kind)
        a, d1 = torch.where(zz < -60, 0.0, torch.where(zz > 60, zz, a)), torch.where(zz.abs() > 60, (zz > 0).double(), d1)
        near(y, a, rounded(a, curve_error(zz, dtype), dtype), "y")
        assert bool(gx.isfinite().all())
        h = passes(lambda x, w, v: layers.gated_feed_forward(x, w, v, torch.eye(w.shape[0], device="cuda", dtype=dtype), kind), [x, w, torch.ones_like(w)], torch.ones(n, w.shape[0], device="cuda", dtype=dtype))
        if n <= 32:
            near(h[0], a, rounded(a, rounded(a, curve_error(zz, dtype), dtype), dtype), "h")


@pytest.mark.gpu
def test_refused_calls(layers):
    x, wg, wu, wd, r, g = gated_inputs(8, 32, 48, 32, torch.bfloat16)
    b = torch.zeros(48, device="cuda", dtype=torch.bfloat16)
    lin, gated, norm = layers.linear, layers.gated_feed_forward, layers.layer_norm
    for call, text in ((lambda: lin(x, wg.half()), "dtype of x"), (lambda: lin(x, wg[:, :16]), "weight must"), (lambda: lin(x, wg, b[:8]), "bias must"), (lambda: lin(x, wg, b.float()), "dtype of x"),
                       (lambda: lin(x, wg, None, None, r), "residual must"), (lambda: lin(x, wg[:0]), "must have rows"), (lambda: lin(x.double(), wg.double()), "fp16, bf16"),
                       (lambda: lin(x, wg.cpu()), "CUDA"), (lambda: lin(x[:, :0], wg[:, :0]), "columns"), (lambda: gated(x, wg, wu[:8], wd), "w_gate and w_up"),
                       (lambda: gated(x, wg, wu, wd[:, :8]), "w_down"), (lambda: gated(x, wg, wu, wd, "silu", b), "residual must"), (lambda: gated(x, wg, wu, wd.float()), "dtype of x"),
                       (lambda: norm(x, b), "must be \\[d\\]"), (lambda: norm(x, b[:32].half()), "dtype of x or float32"), (lambda: norm(x, b[:32], b[:32].float()), "one dtype"),
                       (lambda: norm(torch.zeros(2, 32776, device="cuda")), "32768"), (lambda: norm(x.to(torch.float64)), "fp16, bf16")):
        with pytest.raises(RuntimeError, match=text):
            call()
    import torch.autograd.forward_ad as fad
    for call in (lambda t: lin(t, wg), lambda t: gated(t, wg, wu, wd), lambda t: norm(t)):
        with pytest.raises(RuntimeError, match="traced"):
            torch.jit.trace(call, (x,))
        with fad.dual_level(), pytest.raises(RuntimeError, match="forward-mode"):
            call(fad.make_dual(x, x))


@pytest.mark.gpu
def test_eager_graph_alive_while_a_backward_pass_is_captured(layers):
    # a graph of the same leaves from before stays alive across the capture
    tensors, step = whole(layers, torch.bfloat16, 64)
    leaves = [t.detach().requires_grad_(True) for t in tensors[:4]]
    alive = layers.gated_feed_forward(*leaves)
    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    graph.replay()
    torch.cuda.synchronize()
    for a, b in zip(out, step()):
        assert torch.equal(a, b)
    want = passes(lambda *t: layers.gated_feed_forward(*t), tensors[:4], tensors[-1])
    for a, b in zip(torch.autograd.grad(alive, leaves, tensors[-1]), want[1:]):
        assert torch.equal(a, b)


@pytest.mark.gpu
def test_rows_behind_2_to_31_elements(layers):
    # offsets beyond 32 bits: rows at the end of tall inputs are those of a short call
    d, n = 2048, (1 << 31) // 2048 + 300
    torch.cuda.empty_cache()
    x = torch.zeros(n, d, device="cuda", dtype=torch.bfloat16)
    tail, = inputs([((257, d), 1.0)], torch.bfloat16)
    x[-257:] = tail
    w, = inputs([((8, d), 0.02)], torch.bfloat16, 1)
    want, error = linear_reference(tail, w, None, None, torch.zeros(257, 8, device="cuda", dtype=torch.bfloat16), "gelu", torch.bfloat16)[0]
    near(layers.linear(x, w, activation="gelu")[-257:], want, error, "y")      # the short call shares its sums out, in another order
    assert torch.equal(layers.layer_norm(x)[-257:], layers.layer_norm(tail))
    gated = lambda t: layers.gated_feed_forward(t, w, w, w.T.contiguous())
    assert torch.equal(gated(x)[-257:], gated(tail))


@pytest.mark.gpu
def test_meta_step_of_the_benchmark(layers):
    # the whole second-order step of bench_ttt.py with these operators against its own, as the test of that one compares two attentions
    root = os.path.dirname(PKG_DIR)
    if root not in sys.path:
        sys.path.insert(0, root)
    bt = importlib.import_module("bench_ttt")
    dev = torch.device("cuda")
    attention = importlib.import_module("attention").flash_attention_v7
    for mlp in ("gelu", "gated"):
        cfg, results = dict(bt.SMALL, mlp=mlp), []
        for kind in ("torch", "fused"):
            slow, fast = bt.init_params(cfg, dev, torch.bfloat16, seed=1)
            ids, targets = bt.make_batch(cfg, dev, seed=2)
            out = bt.ttt_step(cfg, slow, fast, ids, targets, lambda q, k, v: attention(q, k, v, cfg["seq"], 0), None, bt.layer_functions(kind))
            out.backward()
            results.append((float(out.detach()), {n: p.grad.float() for n, p in {**slow, **fast}.items()}))
        assert abs(results[0][0] - results[1][0]) < 0.02
        for n, g in results[0][1].items():
            assert torch.allclose(results[1][1][n], g, atol=5e-2 * max(1.0, float(g.abs().max())), rtol=5e-2), n
