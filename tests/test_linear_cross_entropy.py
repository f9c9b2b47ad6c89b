"""Cross entropy of a linear layer without kept logits: refusals (CPU); losses, gradients and the second derivative against
64 bits with bounds derived from the roundings; ignored rows, odd sizes, pieces, shares of k, streams, graphs (GPU)."""
import ctypes
import importlib
import math
import os
import sys

import pytest
import torch

PKG_DIR = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "610sample_b200")


@pytest.fixture(scope="module")
def lce():
    if PKG_DIR not in sys.path:
        sys.path.insert(0, PKG_DIR)
    return importlib.import_module("loss").linear_cross_entropy


@pytest.fixture(scope="module")
def capi():
    return importlib.import_module("610sample_b200.capi")


# ---- CPU ------------------------------------------------------------------------------------------

def _shape(capi, **over):
    d = dict(n=64, d=128, V=1000, dtype=capi.ATTN_BF16, reduction=2, ignore_index=-100)
    d.update(over)
    return capi.LceShape(d["n"], d["d"], d["V"], d["dtype"], d["reduction"], 0, d["ignore_index"])


@pytest.mark.parametrize("over, code, text", [
    (dict(dtype=5), -2, "dtype 5"), (dict(n=-1), -1, "n must"), (dict(n=2 ** 30 + 1), -1, "n must"), (dict(d=0), -1, "d must"),
    (dict(d=2 ** 20 + 1), -1, "d must"), (dict(V=0), -1, "V must"), (dict(V=-7), -1, "V must"), (dict(reduction=3), -1, "reduction"),
])
def test_refused_shapes(capi, over, code, text):
    L, one, s = capi.lib(), ctypes.c_void_p(4096), ctypes.byref(_shape(capi, **over))
    assert L.attn_b200_linear_ce_forward(s, *([one] * 8), None) == code
    assert text in L.attn_b200_last_error().decode()
    assert L.attn_b200_linear_ce_backward(s, *([one] * 9), None) == code
    assert L.attn_b200_linear_ce_forward_scratch_bytes(s) == L.attn_b200_linear_ce_backward_scratch_bytes(s, 1, 1) == 0


def test_refused_pointers(capi):
    L, good, odd = capi.lib(), ctypes.c_void_p(4096), ctypes.c_void_p(4100)
    for i in range(8):
        args = [good] * 8
        args[i] = None
        assert L.attn_b200_linear_ce_forward(ctypes.byref(_shape(capi)), *args, None) == -1
        assert "null" in L.attn_b200_last_error().decode()
    for i in (0, 1, 2, 7):
        args = [good] * 8
        args[i] = odd
        assert L.attn_b200_linear_ce_forward(ctypes.byref(_shape(capi)), *args, None) == -1
        assert "aligned" in L.attn_b200_last_error().decode()
    for i in range(9):
        if i in (6, 7):
            continue
        args = [good] * 9
        args[i] = None
        assert L.attn_b200_linear_ce_backward(ctypes.byref(_shape(capi)), *args, None) == -1
    args = [good] * 6 + [None, None, good]
    assert L.attn_b200_linear_ce_backward(ctypes.byref(_shape(capi)), *args, None) == -1
    assert "neither" in L.attn_b200_last_error().decode()
    assert L.attn_b200_linear_ce_forward(None, *([good] * 8), None) == -1


def test_scratch_does_not_grow_with_the_logits(capi):
    size = lambda n, d, V, dx=1, dw=1, dtype=capi.ATTN_BF16: capi.lib().attn_b200_linear_ce_backward_scratch_bytes(
        ctypes.byref(_shape(capi, n=n, d=d, V=V, dtype=dtype)), dx, dw)
    n, d, V = 16384, 768, 128 * 1024
    assert size(n, d, V) <= (512 << 20) + 4 * n * d + 2 * n * d + 4 * n + (37 << 20) + 4096 < 2 * n * V
    assert size(n, d, V, 1, 0) < size(n, d, V) and size(n, d, V, 0, 1) < size(n, d, V)
    assert size(1, 8, 2) >= 4 + 4 + 16 + 16
    assert capi.lib().attn_b200_linear_ce_forward_scratch_bytes(ctypes.byref(_shape(capi, n=n, d=d, V=V))) <= 8 * n * (V // 256) + 4 * n + 512


def test_python_refusals(lce):
    x, w, y = torch.zeros(4, 8), torch.zeros(10, 8), torch.zeros(4, dtype=torch.long)
    with pytest.raises(ValueError, match="reduction"):
        lce(x, w, y, reduction="median")
    with pytest.raises(RuntimeError, match="shape of x"):
        lce(x, w, y[:3])
    with pytest.raises(RuntimeError, match="CUDA"):
        lce(x, w, y)


# ---- against 64 bits ----------------------------------------------------------------------------------

def reference(x, w, y, g, ignore, reduction):
    """(losses or value, dx, dw) in 64 bits and bounds of the errors.  f = 2^-24; u: half a step of the type that G is rounded
    to (fp32: f).  A logit is a sum of d products: off by e_z = (d + 4) f sum |x w|, the log-sum-exp by the largest e_z of its
    row and a few f of its own size, P relatively by e_P, the sum of both.  G = c (P - onehot): off by c P e_P and rounded, in
    fp16 by at least 2^-25 of the unit (the largest factor over 2^15).  Sums of n products in fp32: n f of the sum of sizes."""
    f, out_u = 2.0 ** -24, torch.finfo(x.dtype).eps / 2
    u = out_u
    n, d = x.shape
    V = w.shape[0]
    x, w = x.double(), w.double()
    keep = (y != ignore)
    at = torch.where(keep, y, 0)
    xk = torch.where(keep[:, None], x, 0.0)
    z = xk @ w.T
    e_z = (xk.abs() @ w.abs().T) * (d + 4) * f
    lse = torch.logsumexp(z, 1, keepdim=True)
    top = z.abs().amax(1, keepdim=True)
    e_lse = e_z.amax(1, keepdim=True) + (V + 24) * f + 8 * f * (lse.abs() + top)
    P = torch.exp(z - lse)
    zy, ezy = z.gather(1, at[:, None]), e_z.gather(1, at[:, None])
    loss = torch.where(keep, (lse - zy)[:, 0], 0.0)
    e_loss = torch.where(keep, (e_lse + ezy + 4 * f * (lse.abs() + zy.abs()))[:, 0], 0.0)
    count = keep.sum()
    share = keep.double() / count if reduction == "mean" else keep.double()
    c = share * g.double()
    onehot = torch.zeros_like(P).scatter_(1, at[:, None], 1.0)
    G = c[:, None] * (P - onehot)
    e_P = e_z + e_lse + 8 * f * (z.abs() + lse.abs()) + 8 * f
    unit = c.abs().amax() / 2 ** 15 if out_u == 2.0 ** -11 else 0.0
    e_G = c.abs()[:, None] * (P * e_P * 1.01 + 4 * f * onehot) + (u + 4 * f) * G.abs() + 2.0 ** -25 * unit
    dx, dw = G @ w, G.T @ xk
    e_dx = (e_G + (V + 8) * f * G.abs()) @ w.abs() + out_u * dx.abs()
    e_dw = (e_G + (n + 8) * f * G.abs()).T @ xk.abs() + out_u * dw.abs()
    if reduction == "none":
        value, e_value = loss, e_loss
    else:
        value, e_value = (loss * share).sum(), (e_loss * share).sum() + f * (loss * share).sum().abs() * 4
    return (value, dx, dw), (e_value + 1e-30, e_dx * 1.02, e_dw * 1.02)


def inputs(n, d, V, dtype, seed=0, spread=2.0, ignored=0.1):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(n, d, generator=g).to(dtype).cuda()
    w = (torch.randn(V, d, generator=g) * spread / math.sqrt(d)).to(dtype).cuda()
    y = torch.randint(0, V, (n,), generator=g)
    y[torch.rand(n, generator=g) < ignored] = -100
    if n:
        y[0] = 0 if n % 2 else V - 1
    return x, w, y.cuda(), (torch.rand(n, generator=g) * 2 - 0.7).cuda()


def both_passes(lce, x, w, y, g, reduction, ignore=-100):
    x, w = x.detach().requires_grad_(True), w.detach().requires_grad_(True)
    out = lce(x, w, y, ignore, reduction)
    return [out.detach(), *torch.autograd.grad(out, (x, w), g)]


def check(lce, n, d, V, dtype, reduction="mean", **kw):
    x, w, y, g = inputs(n, d, V, dtype, **kw)
    g = g if reduction == "none" else torch.tensor(0.7, device="cuda")
    got = both_passes(lce, x, w, y, g, reduction)
    want, bound = reference(x, w, y, g, -100, reduction)
    tiny = torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
    for name, a, b, e in zip(("loss", "dx", "dw"), got, want, bound):
        assert a.shape == b.shape and a.dtype == (torch.float32 if name == "loss" else dtype)
        worst = ((a.double() - b).abs() / (e + (0 if name == "loss" else tiny))).max()
        assert bool(worst <= 1), (name, float(worst))
    assert torch.equal(lce(x, w, y, reduction=reduction), got[0])


SIZES = [(1, 8, 1), (1, 64, 2), (2, 8, 257), (37, 96, 1000), (128, 64, 256), (129, 72, 511), (255, 136, 513), (300, 768, 3001), (513, 320, 1025)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("n, d, V", SIZES)
def test_sizes(lce, dtype, n, d, V):
    check(lce, n, d, V, dtype, ignored=0.1 if n > 4 else 0.0)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("d", [1, 7, 100, 200])
def test_widths_without_tensor_cores(lce, dtype, d):
    check(lce, 140, d, 300, dtype, "none")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("reduction", ["none", "sum", "mean"])
def test_reductions(lce, dtype, reduction):
    check(lce, 200, 128, 700, dtype, reduction)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_peaked_rows(lce, dtype):
    check(lce, 150, 128, 900, dtype, "none", spread=12.0)


@pytest.mark.gpu
@pytest.mark.parametrize("n, d, V", [(33000, 64, 17000), (3000, 128, 100003), (8, 64, 100003), (20000, 8, 3)])
def test_pieces_and_shares_of_k(lce, n, d, V):
    # several pieces of the vocabulary; one row block against a long vocabulary; a long sum over rows for few classes
    check(lce, n, d, V, torch.bfloat16)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("n, d, V", [(5000, 768, 3001), (700, 1000, 20000), (2000, 264, 8192), (9000, 512, 700), (300, 2048, 30000), (16500, 64, 8200)])
def test_tiles_in_several_shares(lce, dtype, n, d, V):
    check(lce, n, d, V, dtype, "none")


@pytest.mark.gpu
def test_pieces_on_cuda_cores(lce):
    check(lce, 33000, 16, 9000, torch.float32)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype, d", [(torch.bfloat16, 64), (torch.float16, 64), (torch.float32, 64), (torch.bfloat16, 60)])
@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_ignored_rows_have_no_influence(lce, dtype, d, bad):
    x, w, y, g = inputs(300, d, 500, dtype, ignored=0.3)
    clean = both_passes(lce, x, w, y, g, "none")
    x[y == -100] = bad
    dirty = both_passes(lce, x, w, y, g, "none")
    for a, b in zip(clean, dirty):
        assert torch.equal(a, b)
    assert not bool(clean[1][y == -100].any()) and not bool(clean[0][y == -100].any())
    assert torch.equal(lce(x, w, y), lce(torch.where((y == -100)[:, None], 0.0, x), w, y))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("reduction", ["none", "sum", "mean"])
def test_a_factor_of_all_rows_is_not_rounded(lce, dtype, reduction):
    # a factor just below the middle of two numbers of the type.  Rounded in every row, it alone would put the gradients off by u = half a
    # step; the roundings of G and of the results are independent and evenly spread, each off by at most u / sqrt(3) in the 2-norm
    u = torch.finfo(dtype).eps / 2
    n = 400
    x, w, y, _ = inputs(n, 128, 2000, dtype, ignored=0.0)
    factor = (1 + u) * (1 - 2.0 ** -20)
    g = torch.full((n,), factor, device="cuda") if reduction == "none" else torch.tensor(factor * (n if reduction == "mean" else 1), device="cuda")
    got = both_passes(lce, x, w, y, g, reduction)
    want, _ = reference(x, w, y, g, -100, reduction)
    for a, b in zip(got[1:], want[1:]):
        assert float((a.double() - b).norm() / b.norm()) <= u * math.sqrt(2 / 3)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype, d", [(torch.bfloat16, 64), (torch.float32, 64), (torch.bfloat16, 60)])
@pytest.mark.parametrize("out", [(0, 300), (300, 600), (3, 20), (500, 900)])
def test_logits_of_minus_infinity_count_nothing(lce, dtype, d, out):
    # classes whose weights are the type's lowest value: their logits overflow to -inf for rows of positive x
    x, w, y, g = inputs(140, d, 900, dtype)
    x = x.abs() + 0.5
    keep = torch.ones(900, dtype=torch.bool, device="cuda")
    keep[out[0]:out[1]] = False
    index = torch.cumsum(keep, 0) - 1
    y = torch.where((y >= 0) & ~keep[y.clamp(min=0)], int(keep.nonzero()[0]), y)
    w[~keep] = torch.finfo(dtype).min
    got = both_passes(lce, x, w, y, g, "none")
    want, bound = reference(x, w[keep], torch.where(y >= 0, index[y.clamp(min=0)], y), g, -100, "none")
    tiny = torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
    assert not bool(got[2][~keep].any())
    for a, b, e in zip((got[0], got[1], got[2][keep]), want, bound):
        assert bool(((a.double() - b).abs() <= e + tiny).all())


@pytest.mark.gpu
def test_nothing_counts(lce):
    x, w, y, g = inputs(20, 32, 50, torch.bfloat16)
    y.fill_(-100)
    assert bool(lce(x, w, y).isnan()) and float(lce(x, w, y, reduction="sum")) == 0.0
    out, dx, dw = both_passes(lce, x, w, y, g, "none")
    assert not bool(out.any()) and not bool(dx.any()) and not bool(dw.any())
    # another class that is ignored
    y.copy_(torch.arange(20) % 4)
    a, b = lce(x, w, y, 2, "none"), lce(x, w, y, -100, "none")
    assert not bool(a[y == 2].any()) and torch.equal(a[y != 2], b[y != 2])


@pytest.mark.gpu
def test_no_such_class_is_not_a_number(lce):
    for dtype in (torch.bfloat16, torch.float32):
        x, w, y, _ = inputs(40, 32, 50, dtype, ignored=0.0)
        y[3], y[7] = 50, -1
        out = lce(x, w, y, reduction="none")
        assert out.isnan().nonzero().flatten().tolist() == [3, 7]
        y[3] = 1 << 40
        assert bool(lce(x, w, y, reduction="none")[3].isnan())


@pytest.mark.gpu
def test_no_rows(lce):
    w = torch.randn(30, 16, device="cuda").bfloat16().requires_grad_(True)
    x = torch.zeros(0, 16, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    y = torch.zeros(0, dtype=torch.long, device="cuda")
    assert lce(x, w, y, reduction="none").shape == (0,)
    s = lce(x, w, y, reduction="sum")
    assert float(s.detach()) == 0.0 and bool(lce(x, w, y).isnan())
    dx, dw = torch.autograd.grad(s, (x, w))
    assert dx.shape == (0, 16) and not bool(dw.any())


@pytest.mark.gpu
def test_layouts_and_shapes(lce):
    x, w, y, g = inputs(24, 64, 100, torch.bfloat16)
    want = both_passes(lce, x, w, y, g, "none")
    xs = torch.empty(24, 130, device="cuda", dtype=torch.bfloat16)[:, 1:129:2]
    xs.copy_(x)
    wt = w.T.contiguous().T
    ys = torch.stack([y, y], 1)[:, 0]
    for got in (both_passes(lce, xs, wt, ys, g, "none"), both_passes(lce, x.view(2, 12, 64), w, y.view(2, 12), g.view(2, 12), "none")):
        for a, b in zip(got, want):
            assert torch.equal(a.reshape(b.shape), b)
    assert torch.equal(lce(x.view(2, 12, 64), w, y.view(2, 12)), lce(x, w, y))
    v = x[0]
    assert lce(v, w, y[0], reduction="none").shape == ()
    # one gradient only
    xl, wl = x.detach().requires_grad_(True), w.detach().requires_grad_(True)
    (dx,) = torch.autograd.grad(lce(xl, w, y, reduction="none"), xl, g)
    (dw,) = torch.autograd.grad(lce(x, wl, y, reduction="none"), wl, g)
    assert torch.equal(dx, want[1]) and torch.equal(dw, want[2])


@pytest.mark.gpu
def test_refused_calls(lce):
    x, w, y, _ = inputs(8, 32, 50, torch.bfloat16)
    for args, text in (((x, w.half(), y), "same dtype"), ((x, w[:, :16], y), "must be"), ((x, w, y.int()), "int64"), ((x.double(), w.double(), y), "fp16, bf16"),
                       ((x, w[:0], y), "not be empty"), ((x, w, y.cpu()), "CUDA"), ((x, w, torch.stack([y, y])), "shape of x")):
        with pytest.raises(RuntimeError, match=text):
            lce(*args)
    with pytest.raises(RuntimeError, match="traced"):
        torch.jit.trace(lambda t: lce(t, w, y), (x,))
    import torch.autograd.forward_ad as fad
    with fad.dual_level(), pytest.raises(RuntimeError, match="forward-mode"):
        lce(fad.make_dual(x, x), w, y)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_captured_and_on_two_streams(lce, dtype):
    x, w, y, g = inputs(300, 64, 700, dtype)
    step = lambda: both_passes(lce, x, w, y, g, "none") + both_passes(lce, x, w, y, None, "mean")
    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for seed in (1, 2):
        for t, s in zip((x, w, y, g), inputs(300, 64, 700, dtype, seed)):
            t.copy_(s)
        graph.replay()
        for a, b in zip(out, step()):
            assert torch.equal(a, b)
    cases = [inputs(300, 64, 5000, dtype, seed) for seed in (3, 4)]
    want = [both_passes(lce, *c, "none") for c in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    for _ in range(4):
        got = []
        for st, c in zip(streams, cases):
            with torch.cuda.stream(st):
                got.append(both_passes(lce, *c, "none"))
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert all(torch.equal(p, q) for p, q in zip(a, b))


@pytest.mark.gpu
@pytest.mark.parametrize("reduction", ["none", "sum", "mean"])
@pytest.mark.parametrize("dtype, tol", [(torch.float32, 2e-5), (torch.bfloat16, 2e-2), (torch.float16, 3e-3)])
def test_second_derivative(lce, dtype, tol, reduction):
    # against the norm of the result; four rounded factors of 2^-8 (2^-11) each, fp32: sums of up to 90 products of sums
    x, w, y, g = inputs(60, 48, 90, dtype, ignored=0.2)
    g = g if reduction == "none" else torch.tensor(1.3, device="cuda")
    u, v, _, _ = inputs(60, 48, 90, dtype, seed=8)
    leaves = [x.requires_grad_(True), w.requires_grad_(True), g.requires_grad_(True)]
    first = torch.autograd.grad(lce(x, w, y, reduction=reduction), (x, w), g, create_graph=True)
    got = torch.autograd.grad(first, leaves, (u, v))
    d = [t.detach().double().requires_grad_(True) for t in leaves]
    out = torch.nn.functional.cross_entropy(d[0] @ d[1].T, y, reduction=reduction)
    f64 = torch.autograd.grad(out, d[:2], d[2], create_graph=True)
    want = torch.autograd.grad(f64, d, (u.double(), v.double()))
    for a, b in zip(got, want):
        assert a.shape == b.shape and float((a.double() - b).norm() / b.norm()) <= tol
    with pytest.raises(RuntimeError, match="third derivative"):
        first = torch.autograd.grad(lce(x, w, y, reduction=reduction), (x, w), g, create_graph=True)
        torch.autograd.grad(first, leaves, (u, v), create_graph=True)


@pytest.mark.gpu
def test_a_factor_of_all_rows_is_not_rounded_in_the_second_derivative(lce):
    # the factor below the middle of two numbers, as above.  H = c P (T - r) and G = c (P - onehot) are rounded element by element, and the
    # results: each off by u / sqrt(3) / m in the mean square, m the mantissa, over [1, 2) 0.408 u; 15 % more for how they really lie
    n, d, V, u = 300, 128, 1500, 2.0 ** -8
    x, w, y, _ = inputs(n, d, V, torch.bfloat16, ignored=0.0)
    tx, tw, _, _ = inputs(n, d, V, torch.bfloat16, seed=8)
    factor = (1 + u) * (1 - 2.0 ** -20)
    leaves = [x.requires_grad_(True), w.requires_grad_(True)]
    first = torch.autograd.grad(lce(x, w, y, reduction="sum"), leaves, torch.tensor(factor, device="cuda"), create_graph=True)
    got = torch.autograd.grad(first, leaves, (tx, tw))
    x, w, tx, tw = (t.detach().double() for t in (x, w, tx, tw))
    P, T = torch.softmax(x @ w.T, 1), tx @ w.T + x @ tw.T
    H = factor * P * (T - (P * T).sum(1, keepdim=True))
    G = factor * (P - torch.nn.functional.one_hot(y, V))
    want = (H @ w + G @ tw, H.T @ x + G.T @ tx)
    squares = lambda a, b: ((a * a) @ (b * b).sum(1)).sum()
    spread = (squares(H, w) + squares(G, tw), squares(H.T, x) + squares(G.T, tx))
    for a, b, e in zip(got, want, spread):
        assert float((a.double() - b).norm()) <= 0.47 * u * float((e + (b * b).sum()).sqrt())


@pytest.mark.gpu
def test_gradient_against_differences(lce):
    # h = 2^-7: truncation h^2 / 6 of a third derivative of the first's size (1e-5), rounding of the sum of 100 losses over 2 h (2e-4)
    x, w, y, _ = inputs(100, 40, 300, torch.float32)
    dx_, dw_, _, _ = inputs(100, 40, 300, torch.float32, seed=5)
    _, dx, dw = both_passes(lce, x, w, y, None, "sum")
    h = 2.0 ** -7
    for grad, direction, moved in ((dx, dx_, lambda s: (x + s * dx_, w)), (dw, dw_, lambda s: (x, w + s * dw_))):
        up, down = (lce(*moved(s * h), y, reduction="none").double().sum() for s in (1, -1))
        want = float((grad.double() * direction.double()).sum())
        assert abs(float(up - down) / (2 * h) - want) <= 5e-3 * float(grad.double().norm() * direction.double().norm()) / math.sqrt(direction.numel()) * 3


@pytest.mark.gpu
def test_meta_step_of_the_benchmark(lce):
    # the whole second-order step with this loss against the one that keeps its logits, as that one's test compares two attentions
    root = os.path.dirname(PKG_DIR)
    if root not in sys.path:
        sys.path.insert(0, root)
    bt = importlib.import_module("bench_ttt")
    cfg, dev = dict(bt.SMALL), torch.device("cuda")
    attention = importlib.import_module("attention").flash_attention_v7
    grads = []
    for loss in (None, lce):
        slow, fast = bt.init_params(cfg, dev, torch.bfloat16, seed=1)
        ids, targets = bt.make_batch(cfg, dev, seed=2)
        out = bt.ttt_step(cfg, slow, fast, ids, targets, lambda q, k, v: attention(q, k, v, cfg["seq"], 0), loss)
        out.backward()
        grads.append((float(out.detach()), {n: p.grad.float() for n, p in {**slow, **fast}.items()}))
    assert abs(grads[0][0] - grads[1][0]) < 0.02
    for n, g in grads[0][1].items():
        assert torch.allclose(grads[1][1][n], g, atol=5e-2 * max(1.0, float(g.abs().max())), rtol=5e-2), n


def second_of(lce, x, w, y, g, u, v, reduction):
    """((d/dg, d/dx, d/dw) of <first gradients, (u, v)>, the same in 64 bits)"""
    leaves = [t.detach().requires_grad_(True) for t in (x, w, g)]
    first = torch.autograd.grad(lce(leaves[0], leaves[1], y, reduction=reduction), leaves[:2], leaves[2], create_graph=True)
    got = torch.autograd.grad(first, leaves, (u, v))
    d = [t.detach().double().requires_grad_(True) for t in leaves]
    f64 = torch.autograd.grad(torch.nn.functional.cross_entropy(d[0] @ d[1].T, y, reduction=reduction), d[:2], d[2], create_graph=True)
    return got, torch.autograd.grad(f64, d, (u.double(), v.double()))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype, tol", [(torch.float32, 2e-5), (torch.float16, 3e-3)])
def test_second_derivative_under_the_callers_precision(lce, dtype, tol):
    # the tolerances of test_second_derivative, whatever the process allows its own products
    matmul = torch.backends.cuda.matmul
    x, w, y, _ = inputs(300, 256, 700, dtype, ignored=0.2)
    u, v, _, _ = inputs(300, 256, 700, dtype, seed=8)
    g = torch.tensor(1.3, device="cuda")
    before = torch.get_float32_matmul_precision(), matmul.allow_fp16_accumulation, matmul.allow_fp16_reduced_precision_reduction, torch.backends.cuda.preferred_blas_library()
    try:
        for precision in ("high", "medium"):
            for library in ("cublas", "cublaslt"):
                torch.set_float32_matmul_precision(precision)
                torch.backends.cuda.preferred_blas_library(library)
                matmul.allow_fp16_accumulation = matmul.allow_fp16_reduced_precision_reduction = True
                for a, b in zip(*second_of(lce, x, w, y, g, u, v, "mean")):
                    assert float((a.double() - b).norm() / b.norm()) <= tol, (precision, library)
                assert torch.get_float32_matmul_precision() == precision and matmul.allow_fp16_accumulation      # left as they were
    finally:
        torch.set_float32_matmul_precision(before[0])
        matmul.allow_fp16_accumulation, matmul.allow_fp16_reduced_precision_reduction = before[1:3]
        torch.backends.cuda.preferred_blas_library(before[3])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype, tol", [(torch.float32, 2e-5), (torch.float16, 3e-3)])
def test_second_derivative_under_autocast(lce, dtype, tol):
    x, w, y, _ = inputs(300, 256, 700, dtype, ignored=0.2)
    u, v, _, _ = inputs(300, 256, 700, dtype, seed=8)
    with torch.autocast("cuda", torch.bfloat16):
        got = second_of(lce, x, w, y, torch.tensor(1.3, device="cuda"), u, v, "mean")[0]
    want = second_of(lce, x, w, y, torch.tensor(1.3, device="cuda"), u, v, "mean")[1]
    for a, b in zip(got, want):
        assert float((a.double() - b).norm() / b.norm()) <= tol


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_no_such_class_is_not_a_number_in_the_second_derivative(lce, dtype):
    # as the loss and the first gradients: the row's, and all that sums over it
    for wrong in (50, -1, 1 << 40):
        x, w, y, g = inputs(40, 32, 50, dtype, ignored=0.2)
        y[3] = wrong
        leaves = [t.detach().requires_grad_(True) for t in (x, w, g)]
        first = torch.autograd.grad(lce(leaves[0], leaves[1], y, reduction="none"), leaves[:2], leaves[2], create_graph=True)
        assert first[0].isnan().any(1).nonzero().flatten().tolist() == [3] and bool(first[1].isnan().any())
        gx, gw, gg = torch.autograd.grad(first, leaves, [t.detach() for t in inputs(40, 32, 50, dtype, seed=8)[:2]])
        assert gx.isnan().all(1).nonzero().flatten().tolist() == [3] and gg.isnan().nonzero().flatten().tolist() == [3] and bool(gw.isnan().all())
        assert not bool(gx[y == -100].any()) and not bool(gg[y == -100].any())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype, d", [(torch.bfloat16, 256), (torch.float16, 256), (torch.float32, 256), (torch.bfloat16, 252)])
@pytest.mark.parametrize("low, high", [(0.5, 8.0), (8.0, 40.0), (40.0, 500.0), (500.0, 30000.0)])
def test_losses_of_sure_rows(lce, dtype, d, low, high):
    # logits of 0 but for the target's, all exact: log(1 + (V - 1) e^-top), near 0 beside logits that are not.  A term of the sum goes through up to five
    # exponentials of 2^-22 each: its own, the two moves of its part's reference (from 0 or -7 to the target), the joins of halves and of tiles; the sums of 256
    # terms and the logarithm are within 2^-22 beside them, and the difference of target and maximum within 2^-22 of itself
    w = torch.eye(d, device="cuda", dtype=dtype)
    y = torch.arange(300, device="cuda") % d
    top = torch.linspace(low, high, 300, device="cuda").to(dtype).unsqueeze(1)
    x = w[y] * top
    for z in (x, x - w[(y + 1) % d] * 7):      # another class below the others
        got = lce(z, w, y, reduction="none").double()
        want = torch.nn.functional.cross_entropy(z.double() @ w.double().T, y, reduction="none")
        assert bool((got >= 0).all()) and float(((got - want).abs() / (6 * 2.0 ** -22 + 2.0 ** -22 * want)).max()) <= 1, float((got - want).abs().max())
    # and of rows that are sure of another class: top, with the same share of its own size
    got = lce(x, w, (y + 3) % d, reduction="none").double()
    want = torch.nn.functional.cross_entropy(x.double() @ w.double().T, (y + 3) % d, reduction="none")
    assert float(((got - want).abs() / (6 * 2.0 ** -22 + 2.0 ** -22 * want)).max()) <= 1


@pytest.mark.gpu
@pytest.mark.parametrize("dtype, d", [(torch.bfloat16, 256), (torch.float16, 256), (torch.float32, 256), (torch.bfloat16, 252)])
@pytest.mark.parametrize("low, high", [(8.0, 24.0), (24.0, 100.0), (100.0, 500.0), (500.0, 30000.0)])
def test_gradients_of_sure_rows(lce, dtype, d, low, high):
    # the rows above; with W = 1, dx is G.  At the target G = -(V - 1) e^-top / (1 + ...), of which the log-sum-exp, rounded once, knows half a step (top 2^-24
    # and less), beside the 2^-22 of the exponential that is the target's share of its sum; it is top itself where both are below a quarter of a step, from 24
    # on.  The exponential of the difference is off by 2^-22
    w = torch.eye(d, device="cuda", dtype=dtype)
    y = torch.arange(300, device="cuda") % d
    top = torch.linspace(low, high, 300, device="cuda").to(dtype).unsqueeze(1)
    x = w[y] * top
    dx = both_passes(lce, x, w, y, torch.ones(300, device="cuda"), "none")[1].double()
    want = torch.softmax(x.double() @ w.double().T, 1) - w[y].double()
    bound = 2.0 ** -22 + (top.double() * 2.0 ** -24 + 2.0 ** -22 if low < 24 else 0.0) + (torch.finfo(dtype).eps + 2.0 ** -20) * want.abs()
    assert float(((dx - want).abs() / bound).max()) <= 1, float((dx - want).abs().max())
