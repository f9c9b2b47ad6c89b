"""Layer operators at the edges: results changed in place, exact zeros and projections beyond the range of f16 in gated blocks,
NaN in weights, second derivatives that are captured, of many tiles and of views, the benchmark's meta-step by relative size."""
import ctypes
import importlib
import json
import math
import os
import subprocess
import sys

import pytest
import torch

from test_layers import (ACTIVATIONS, F32, HALF, PKG_DIR, SECOND, TYPES, capi, close, curve, curve_error, define_act, gated_inputs, inputs, layers, mm, near, norm_inputs,  # noqa: F401
                         passes, rounded, second)

CURVES = [a for a in ACTIVATIONS if a is not None]


# ---- CPU ------------------------------------------------------------------------------------------

def test_scratch_of_calls_without_rows_or_columns(capi):
    L = capi.lib()
    for dtype in (capi.ATTN_F16, capi.ATTN_BF16, capi.ATTN_F32):
        for n, m in ((0, 0), (0, 16), (16, 0)):
            for pass_ in range(3):
                e = capi.Elements()
                e.n, e.m, e.dtype, e.activation, e.pass_ = n, m, dtype, 1, pass_
                least = L.attn_b200_elements_scratch_bytes(ctypes.byref(e))
                assert least == (4 * m if n == 0 else 0)
            for form in range(3):
                for rows, cols, k in ((n, m, 64), (n, m, 0), (64, n, m), (n, 64, m)):
                    if k == 0 and rows and cols:
                        continue
                    c = capi.Products()
                    c.dtype, c.form, c.count = dtype, form, 1
                    p = c.product[0]
                    p.rows, p.cols, p.k, p.pairs = rows, cols, k, 1
                    if rows == 0 or cols == 0:
                        assert L.attn_b200_products_scratch_bytes(ctypes.byref(c)) == 0
        s = capi.NormShape(0, 64, dtype, 0, 1e-5, 0, 64, 64, 64)
        assert L.attn_b200_layer_norm_backward_scratch_bytes(ctypes.byref(s)) == 0


def test_which_calls_are_of_few_rows(capi):
    # tiles of a long sum are shared out and need scratch, few rows do not
    def scratch(rows, k, cols):
        c = capi.Products()
        c.dtype, c.form, c.count = capi.ATTN_BF16, 0, 1
        p = c.product[0]
        p.rows, p.cols, p.k, p.pairs = rows, cols, k, 1
        return capi.lib().attn_b200_products_scratch_bytes(ctypes.byref(c))

    assert scratch(16, 4096, 6144) == 0 and scratch(17, 4096, 6144) > 0
    assert scratch(32, 8192, 2048) == 0 and scratch(33, 8192, 2048) > 0


# ---- no rows ---------------------------------------------------------------------------------------------

@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_norm_of_no_rows_without_parameters(layers, dtype):
    # gradients without elements have no address; both orders
    x, g = (torch.zeros(2, 0, 16, device="cuda", dtype=dtype, requires_grad=True) for _ in range(2))
    first, = torch.autograd.grad(layers.layer_norm(x), x, g, create_graph=True)
    assert first.shape == x.shape
    for t in torch.autograd.grad(first, [x, g], torch.zeros_like(x)):
        assert t.shape == x.shape


# ---- results belong to the caller -----------------------------------------------------------------------

def calls(layers, dtype, lead, k, m):
    """(operator, leaves, cotangent) of rows with these leading axes"""
    n = math.prod(lead)
    x, w, b, r, g = inputs([((n, k), 1.0), ((m, k), 0.2), ((m,), 0.5), ((n, m), 1.0), ((n, m), 1.0)], dtype)
    wg, wu, wd = inputs([((m, k), 0.2), ((m, k), 0.2), ((k, m), 0.2)], dtype, 1)
    at = lambda t: t.reshape(*lead, t.shape[-1])
    x, r, g, gx = at(x), at(r), at(g), at(inputs([((n, k), 1.0)], dtype, 2)[0])
    return [(lambda x, w: layers.linear(x, w), [x, w], g), (lambda x, w, b, r: layers.linear(x, w, b, "gelu", r), [x, w, b, r], g),
            (lambda x, a, b, c: layers.gated_feed_forward(x, a, b, c), [x, wg, wu, wd], gx), (lambda x: layers.layer_norm(x), [x], gx)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("lead", [(), (1,), (5,), (2, 3), (1, 1), (4, 50), (0,), (2, 0)])
@pytest.mark.parametrize("k, m", [(16, 24), (24, 21), (13, 16)])
def test_results_may_be_changed_in_place(layers, dtype, lead, k, m):
    # as those of PyTorch's own operators: y, then 2 (y + 1), whose gradients are those of twice the cotangent
    for call, leaves, g in calls(layers, dtype, lead, k, m):
        want = passes(call, leaves, 2 * g)
        t = [v.detach().requires_grad_(True) for v in leaves]
        y = call(*t)
        assert torch.equal(y, want[0]) and not y._is_view()
        y += 1
        y.mul_(2)
        assert torch.equal(y, (want[0] + 1) * 2)
        for a, b in zip(torch.autograd.grad(y, t, g), want[1:]):
            assert torch.equal(a, b)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_gradients_are_not_their_cotangents(layers, dtype):
    # one row: the bias' cotangent is a gradient of the row's, in memory of its own
    x, w, b, g = inputs([((1, 16), 1.0), ((24, 16), 0.2), ((24,), 0.5), ((1, 24), 1.0)], dtype)
    t = [v.detach().requires_grad_(True) for v in (x, w, b, g)]
    grad_b = torch.autograd.grad(layers.linear(*t[:3]), t[2], t[3], create_graph=True)[0]
    u, = inputs([((24,), 1.0)], dtype, 1)
    got, = torch.autograd.grad(grad_b, t[3], u)
    assert torch.equal(got[0], u) and got.data_ptr() != u.data_ptr()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_negations_that_have_not_been_carried_out(layers, dtype):
    # views with the negative bit, as the imaginary part of a conjugate is: the results of the negated tensors
    views = [lambda t: torch._neg_view(t)] + [lambda t: torch.complex(torch.zeros_like(t), t).conj().imag] * (dtype == torch.float32)
    for k, m in ((16, 24), (13, 1)):
        for call, leaves, g in calls(layers, dtype, (9,), k, m):
            for view in views:
                want = passes(call, [-t for t in leaves], -g)
                t = [v.detach().requires_grad_(True) for v in leaves]
                y = call(*[view(v) for v in t])
                assert torch.equal(y, want[0])
                for a, b in zip(torch.autograd.grad(y, t, view(g)), want[1:]):
                    assert torch.equal(a, -b)


@pytest.mark.gpu
def test_autocast_casts_nothing(layers):
    x, wg, wu, wd, r, g = gated_inputs(9, 32, 48, 32, torch.float32)
    nw = torch.ones(32, device="cuda")
    for call, leaves in ((lambda *t: layers.gated_feed_forward(*t), [x, wg, wu, wd]), (lambda *t: layers.linear(*t), [x, wd[:, :32].contiguous()]), (lambda *t: layers.layer_norm(*t), [x, nw])):
        want = passes(call, leaves, g)
        with torch.autocast("cuda", torch.bfloat16):
            for a, b in zip(passes(call, leaves, g), want):
                assert a.dtype == torch.float32 and torch.equal(a, b)
            if leaves[1].dim() == 2:
                with pytest.raises(RuntimeError, match="dtype of x"):
                    call(x.bfloat16(), *leaves[1:])


# ---- gated blocks: zeros, and projections beyond 65504 -----------------------------------------------------

@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("kind", ACTIVATIONS)
@pytest.mark.parametrize("n", [5, 20, 150])
def test_zeros_stay_zeros(layers, dtype, kind, n):
    # cotangents of the size that loss scaling gives them: a zero that came back as anything else would show
    x, wg, wu, wd, r, g = gated_inputs(n, 64, 96, 64, dtype)
    g = g * 1024
    call = lambda x, a, b, c: layers.gated_feed_forward(x, a, b, c, kind)
    none = torch.zeros_like(wu)
    # without w_up: u = 0, so x and w_gate have no influence
    _, gx, gg, gu, gd = passes(call, [x, wg, none, wd], g)
    assert not bool(gx.any()) and not bool(gg.any()) and bool(gu.any()) and not bool(gd.any())
    # rows of zeros: z = u = 0
    rows = torch.arange(n, device="cuda") % 3 == 0
    blank = torch.where(rows[:, None], torch.zeros_like(x), x)
    y, gx, _, _, _ = passes(call, [blank, wg, wu, wd], g)
    assert not bool(y[rows].any()) and not bool(gx[rows].any()) and bool(gx[~rows].any())
    # second derivative along x, without w_up: the tangent of u is 0 too, and what reaches w_gate has it as a factor
    t = [v.detach().requires_grad_(True) for v in (x, wg, none, wd)]
    grad_x, = torch.autograd.grad(call(*t), t[0], g, create_graph=True)
    assert not bool(torch.autograd.grad(grad_x, t[1], torch.ones_like(x))[0].any())


def gated_bounds(x, wg, wu, wd, g, kind, dtype):
    """(y, gx, gg, gu, gd) in 64 bits, each with what roundings may make of it.  z and u are kept with 11 bits of mantissa (bf16) and 13 (f16), to the nearest; below
    2^-15 f16's are 2^-28 apart."""
    x, wg, wu, wd, g = (t.double() for t in (x, wg, wu, wd, g))
    zero = torch.zeros_like
    z, ez = mm(x, zero(x), wg.T, zero(wg.T), x.shape[1])
    u, eu = mm(x, zero(x), wu.T, zero(wu.T), x.shape[1])
    a, d1, _ = curve(z, kind)
    own = curve_error(z, dtype)
    own_slope = curve_error(z, dtype) - 4 * F32 * z.abs() + 4 * F32
    change = torch.where(z.abs() > 60, 0.0, 1.25)      # |a''| <= 1.25, and far out the slope does not change
    h = a * u
    eh = rounded(h, (ez * 1.2 + own) * (u.abs() + eu) + a.abs() * eu + 4 * F32 * h.abs(), dtype)
    y, ey = mm(h, eh, wd.T, zero(wd.T), wd.shape[1])
    step, tiny = {torch.bfloat16: (2.0 ** -12, 0.0), torch.float16: (2.0 ** -14, 2.0 ** -29), torch.float32: (0.0, 0.0)}[dtype]
    kz, ku = ez + step * (z.abs() + ez) + tiny, eu + step * (u.abs() + eu) + tiny
    ea, ed = kz * 1.2 + own, kz * change + own_slope
    gh, egh = mm(g, zero(g), wd, zero(wd), wd.shape[0])
    dz, du = gh * d1 * u, gh * a
    edz = rounded(dz, egh * (d1 * u).abs() + (gh.abs() + egh) * (ed * (u.abs() + ku) + d1.abs() * ku) + 6 * F32 * dz.abs(), dtype)
    edu = rounded(du, egh * a.abs() + (gh.abs() + egh) * ea + 4 * F32 * du.abs(), dtype)
    x1, e1 = mm(dz, edz, wg, zero(wg), 2 * wg.shape[0])
    x2, e2 = mm(du, edu, wu, zero(wu), 2 * wg.shape[0])
    results = [(y, ey), (x1 + x2, e1 + e2), mm(dz.T, edz.T, x, zero(x), x.shape[0]), mm(du.T, edu.T, x, zero(x), x.shape[0]), mm(g.T, zero(g.T), h, eh, x.shape[0])]
    return [(v, rounded(v, e, dtype)) for v, e in results]


def far_inputs(n, dtype, d=24, f=48, seed=0):
    """A block whose rows' first element, about 4, goes into u alone for half of the inner columns (u about 1e5 or -1e5 beside z about -2), and into z alone
    for the others (z about 1e5 or -1e5 beside a small u), so that h stays below 65504"""
    x, wg, wu, wd, g = inputs([((n, d), 0.4), ((f, d), 0.05), ((f, d), 0.03), ((d, f), 2.0 ** -7), ((n, d), 2.0 ** -5)], dtype, seed)
    v = torch.Generator().manual_seed(seed + 1)
    x[:, 0] = (3.8 + 0.4 * torch.rand(n, generator=v)).to(dtype).cuda()
    x[:, 1] = 1
    far = torch.where(torch.rand(f, generator=v) < 0.5, -25000.0, 25000.0).to(dtype).cuda()
    half = f // 2
    wu[:half, 0], wg[:half, 0], wg[:half, 1] = far[:half], 0, -2
    wg[half:, 0], wu[half:, 0] = far[half:], 0
    return x, wg, wu, wd, g


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("kind", CURVES)
@pytest.mark.parametrize("n", [5, 20, 150])
def test_projections_beyond_65504(layers, dtype, kind, n):
    x, wg, wu, wd, g = far_inputs(n, dtype)
    call = lambda *t: layers.gated_feed_forward(*t, kind)
    want = gated_bounds(x, wg, wu, wd, g, kind, dtype)
    z, u = x.double() @ wg.double().T, x.double() @ wu.double().T
    assert float(z.abs().max()) > 7e4 and float(u.abs().max()) > 7e4 and float((curve(z, kind)[0] * u).abs().max()) < 65504
    for name, a, (v, e) in zip(("y", "gx", "gg", "gu", "gd"), passes(call, [x, wg, wu, wd], g), want):
        near(a, v, e, name)
    # second derivatives: the halves of the weights' gradients by themselves, which have different sizes
    tangents = inputs([((n, 24), 0.4), ((48, 24), 0.03), ((48, 24), 0.03), ((24, 48), 2.0 ** -7)], dtype, 3)
    define = lambda x, a, b, c: (define_act(x @ a.T, kind) * (x @ b.T)) @ c.T
    got, ref = second(call, [x, wg, wu, wd], g, tangents, define)
    for a, b in zip(got, ref):
        for p, q in ((a[:24], b[:24]), (a[24:], b[24:])) if b.shape[0] == 48 else ((a, b),):
            close([p], [q], dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("n", [5, 150])
def test_projections_beyond_what_is_kept(layers, n):
    # f16, u = 20000 x 60000^2 > 2^46 beside z = -40: h = -0.012, and gradients that say that they are lost
    x, wu = (torch.full(s, 60000.0, device="cuda", dtype=torch.float16) for s in ((n, 20000), (8, 20000)))
    wg = torch.zeros_like(wu)
    wg[:, 0] = -40 / 60000
    wd, g = torch.eye(8, device="cuda", dtype=torch.float16), torch.ones(n, 8, device="cuda", dtype=torch.float16)
    y, _, gg, _, _ = passes(lambda *t: layers.gated_feed_forward(*t), [x, wg, wu, wd], g)
    z = -60000.0 * -float(wg[0, 0])
    want = z / (1 + math.exp(-z)) * 20000 * 60000.0 ** 2
    assert bool(((y.double() - want).abs() <= 1e-3 * abs(want)).all()) and bool(gg.isnan().all())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("kind", CURVES)
@pytest.mark.parametrize("n", [401, 21])
def test_far_arguments_and_slopes(layers, dtype, kind, n):
    # one input times one weight: z over a wide range, u = 2^-15 z, results and all gradients
    top = 32000 if dtype == torch.float16 else 1e15
    z = torch.logspace(-4, math.log10(top), n // 2)
    x = torch.cat([-z, torch.zeros(1), z]).to(dtype).cuda()[:, None]
    w, v = torch.ones(8, 1, device="cuda", dtype=dtype), torch.full((8, 1), 2.0 ** -15, device="cuda", dtype=dtype)
    eye, g = torch.eye(8, device="cuda", dtype=dtype), torch.full((n, 8), 2.0 ** -3, device="cuda", dtype=dtype)
    want = gated_bounds(x, w, v, eye, g, kind, dtype)
    got = passes(lambda *t: layers.gated_feed_forward(*t, kind), [x, w, v, eye], g)
    for name, a, (t, e) in zip(("y", "gx", "gg", "gu", "gd"), got, want):
        if name in ("y", "gx") or dtype == torch.bfloat16:      # sums of squares leave the range of f16
            near(a, t, e, name)
    # a linear layer: eight equal terms make the slope, which is 0 or 1 far out
    gx = passes(lambda x, w: layers.linear(x, w, activation=kind), [x, w], g)[1]
    zz = x.double()
    slope = torch.where(zz.abs() > 60, (zz > 0).double(), curve(zz, kind)[1])
    kept = rounded(zz.clamp(-60, 60), 0 * zz, torch.float16)
    error = torch.where(zz.abs() > 60, 0.0, curve_error(zz, dtype) + 1.25 * kept)
    near(gx, slope, rounded(slope, rounded(slope, error + 12 * F32, dtype), dtype), "slope")


# ---- NaN ----------------------------------------------------------------------------------------------

@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("kind", CURVES)
@pytest.mark.parametrize("n", [5, 20, 150])
def test_nan_in_a_weight_reaches_its_gradients(layers, dtype, kind, n):
    # a row of a weight: the inner column that it makes is NaN, with its gradients, and the other columns' gradients are as they were
    x, wg, wu, wd, r, g = gated_inputs(n, 64, 96, 64, dtype)
    w, b, gf = inputs([((96, 64), 0.2), ((96,), 0.3), ((n, 96), 1.0)], dtype, 4)
    others = torch.arange(96, device="cuda") != 40
    spoil = lambda t: torch.where(others[:, None], t, torch.full_like(t, float("nan")))

    def look(grad, clean, lost):
        assert torch.equal(grad[others], clean[others])
        assert bool(grad[40].isnan().all()) if lost else torch.equal(grad[40], clean[40])

    call = lambda x, w, b: layers.linear(x, w, b, kind)
    clean, soiled = passes(call, [x, w, b], gf), passes(call, [x, spoil(w), b], gf)
    look(soiled[0].T, clean[0].T, True)
    assert bool(soiled[1].isnan().all())
    look(soiled[2], clean[2], True)
    look(soiled[3], clean[3], True)
    call = lambda *t: layers.gated_feed_forward(*t, kind)
    clean = passes(call, [x, wg, wu, wd], g)
    for weights, gate_lost, up_lost in (([spoil(wg), wu], True, True), ([wg, spoil(wu)], True, False)):
        soiled = passes(call, [x, *weights, wd], g)
        assert bool(soiled[0].isnan().all()) and bool(soiled[1].isnan().all())
        look(soiled[2], clean[2], gate_lost)
        look(soiled[3], clean[3], up_lost)
        look(soiled[4].T, clean[4].T, True)


# ---- second derivatives as they are called ---------------------------------------------------------------

def second_steps(layers, dtype, n=150, d=72, f=104, seed=0):
    """(tensors, a function that gives all second derivatives of the three operators)"""
    x, wg, wu, wd, r, g = gated_inputs(n, d, f, d, dtype, seed)
    w, b, gf = inputs([((f, d), 0.2), ((f,), 0.3), ((n, f), 1.0)], dtype, seed + 40)
    nw, nb = inputs([((d,), 0.3), ((d,), 0.3)], dtype, seed + 41)
    u = gated_inputs(n, d, f, d, dtype, seed + 42)
    uw, ub, uf = inputs([((f, d), 0.2), ((f,), 0.3), ((d,), 0.3)], dtype, seed + 43)
    tensors = [x, wg, wu, wd, g, w, b, gf, nw, nb, *u[:4], uw, ub, uf]

    def step(x, wg, wu, wd, g, w, b, gf, nw, nb, ux, ug, uu, ud, uw, ub, uf):
        out = []
        for call, leaves, up, along in ((lambda *t: layers.gated_feed_forward(*t), [x, wg, wu, wd], g, [ux, ug, uu, ud]),
                                        (lambda *t: layers.linear(*t, "gelu"), [x, w, b], gf, [ux, uw, ub]), (lambda *t: layers.linear(*t), [x, w, b], gf, [ux, uw, ub]),
                                        (lambda *t: layers.layer_norm(*t), [x, nw, nb], g, [ux, uf, uf])):
            t = [v.detach().requires_grad_(True) for v in leaves + [up]]
            first = torch.autograd.grad(call(*t[:-1]), t[:-1], t[-1], create_graph=True)
            out += [v for v in torch.autograd.grad(first, t, along, allow_unused=True) if v is not None]
        return out

    return tensors, step


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n", [3, 150])
def test_captured_second_derivatives(layers, dtype, n):
    tensors, step = second_steps(layers, dtype, n)
    step(*tensors)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(*tensors)
    for seed in (1, 2):
        for t, s in zip(tensors, second_steps(layers, dtype, n, seed=seed)[0]):
            t.copy_(s)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(out, step(*tensors)):
            assert torch.equal(a, b)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n", [6, 150])
def test_second_derivatives_of_views(layers, dtype, n):
    # cotangents and inputs that are slices of wider rows (where 16 bytes divide their starts, the norm reads them as it reads dense ones), transposed, expanded
    tensors, step = second_steps(layers, dtype, n)
    plain = step(*tensors)

    def inside(t):
        wide = torch.full((t.shape[0], t.shape[1] + 16), float("nan"), device="cuda", dtype=dtype)
        wide[:, 8:8 + t.shape[1]] = t
        return wide[:, 8:8 + t.shape[1]]

    for view in (inside, lambda t: t.T.contiguous().T):
        for a, b in zip(step(*[view(t) if t.dim() == 2 else t for t in tensors]), plain):
            assert torch.equal(a, b)
    spread = lambda t: t[:1].expand(t.shape) if t.dim() == 2 else t[:1].expand(t.shape)
    along = range(10, len(tensors))
    for a, b in zip(step(*[spread(t) if i in along else t for i, t in enumerate(tensors)]), step(*[spread(t).contiguous() if i in along else t for i, t in enumerate(tensors)])):
        assert torch.equal(a, b)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", HALF)
def test_second_derivatives_of_many_tiles(layers, dtype):
    # several rounds of tiles, and sums over the rows that are shared out
    n, k, m = 2500, 520, 2600
    leaves = inputs([((n, k), 1.0), ((m, k), 1.5 / math.sqrt(k)), ((m,), 0.5)], dtype)
    g, = inputs([((n, m), 1.0)], dtype, 5)
    tangents = inputs([((n, k), 1.0), ((m, k), 1 / math.sqrt(k)), ((m,), 1.0)], dtype, 6)
    close(*second(lambda x, w, b: layers.linear(x, w, b, "silu"), leaves, g, tangents, lambda x, w, b: define_act(x @ w.T + b, "silu")), dtype)
    x, wg, wu, wd, r, g = gated_inputs(n, k, 1304, k, dtype)
    tangents = gated_inputs(n, k, 1304, k, dtype, 9)[:4]
    close(*second(lambda *t: layers.gated_feed_forward(*t, "gelu"), [x, wg, wu, wd], g, tangents, lambda x, a, b, c: (define_act(x @ a.T, "gelu") * (x @ b.T)) @ c.T), dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d, f", [(64, 96), (61, 99)])
def test_saved_tensors_that_move(layers, dtype, d, f):
    # what is kept goes to the host and comes back, with other strides
    x, wg, wu, wd, r, g = gated_inputs(150, d, f, d, dtype)
    w, gf = inputs([((f, d), 0.2), ((150, f), 1.0)], dtype, 4)
    for call, leaves, up in ((lambda *t: layers.gated_feed_forward(*t), [x, wg, wu, wd], g), (lambda *t: layers.linear(*t, None, "gelu"), [x, w], gf),
                             (lambda t: layers.layer_norm(t), [x], g)):
        want = passes(call, leaves, up)
        with torch.autograd.graph.save_on_cpu():
            got = passes(call, leaves, up)
        for a, b in zip(got, want):
            assert torch.equal(a, b)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("k, m", [(64, 96), (61, 99)])
def test_inputs_changed_before_the_backward_are_noticed(layers, dtype, k, m):
    for call, leaves, up in calls(layers, dtype, (9,), k, m):
        for i in range(min(2, len(leaves))):
            t = [v.detach().clone().requires_grad_(True) for v in leaves]
            y = call(*t)
            with torch.no_grad():
                t[i].mul_(2)
            with pytest.raises(RuntimeError, match="inplace"):
                torch.autograd.grad(y, t, up)


# ---- the benchmark's step ----------------------------------------------------------------------------------

@pytest.mark.gpu
@pytest.mark.parametrize("mlp", ["gelu", "gated"])
def test_meta_step_by_relative_size(layers, mlp):
    # every parameter's gradient in the 2-norm.  float32: sums of up to 256 products are off by 256 f of their sizes at most, in about 60 products one behind the other: 1e-3.
    # bf16: the operators round less often than PyTorch's chain of separate operations, so they are no further from float32 than twice what that chain is
    root = os.path.dirname(PKG_DIR)
    if root not in sys.path:
        sys.path.insert(0, root)
    bt = importlib.import_module("bench_ttt")
    attention = importlib.import_module("attention").flash_attention_v7
    cfg = dict(bt.SMALL, mlp=mlp)
    dev = torch.device("cuda")

    def gradients(kind, dtype):
        slow, fast = bt.init_params(cfg, dev, torch.bfloat16, seed=1)
        slow, fast = ({n: p.detach().to(dtype).requires_grad_(True) for n, p in group.items()} for group in (slow, fast))
        ids, targets = bt.make_batch(cfg, dev, seed=2)
        bt.ttt_step(cfg, slow, fast, ids, targets, lambda q, k, v: attention(q, k, v, cfg["seq"], 0), None, bt.layer_functions(kind)).backward()
        return {n: p.grad.double() for n, p in {**slow, **fast}.items()}

    want = gradients("torch", torch.float32)
    away = lambda got: {n: float((got[n] - want[n]).norm() / want[n].norm()) for n in want}
    assert all(float(v.norm()) > 0 for v in want.values())
    for n, e in away(gradients("fused", torch.float32)).items():
        assert e <= 1e-3, (n, e)
    chain = away(gradients("torch", torch.bfloat16))
    for n, e in away(gradients("fused", torch.bfloat16)).items():
        assert e <= 2 * chain[n], (n, e, chain[n])


@pytest.mark.gpu
@pytest.mark.parametrize("mlp", ["gelu", "gated"])
def test_the_benchmark_says_what_it_ran(mlp):
    root = os.path.dirname(PKG_DIR)
    run = subprocess.run([sys.executable, os.path.join(root, "bench_ttt.py"), "--small", "--steps", "1", "--warmup", "1", "--layers", "fused", "--mlp", mlp],
                         capture_output=True, text=True, timeout=300, cwd=root)
    assert run.returncode == 0, run.stderr[-2000:]
    config = json.loads(run.stdout.strip().splitlines()[-1])["config"]
    assert config["layers"] == 2 and config["layer_operators"] == "fused" and config.get("mlp", "gelu") == mlp
