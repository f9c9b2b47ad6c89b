"""Attention on packed batches: refusals (CPU), the plan, both passes against a plain implementation in 64 bits
with bounds derived from the roundings, isolation of the sequences, strides, streams, graphs, the second
derivative (GPU)."""
import ctypes
import importlib
import math
import os
import subprocess
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
def capi():
    return importlib.import_module("610sample_b200.capi")


def offsets(lens, front=0):
    cu = [front]
    for n in lens:
        cu.append(cu[-1] + n)
    return cu


# ---- CPU ------------------------------------------------------------------------------------------

def _shape(capi, **over):
    s = capi.PackedShape()
    d = dict(n_tok=256, n_seq=2, q_heads=4, kv_heads=2, D=64, window_size=2 ** 31 - 1, dtype=capi.ATTN_BF16)
    d.update({k: v for k, v in over.items() if k in d})
    for k, v in d.items():
        setattr(s, k, v)
    for i, h in enumerate((4, 2, 2, 4)):
        s.row_stride[i], s.head_stride[i] = over.get("row", h * 64), over.get("head", 64)
    return s


@pytest.mark.parametrize("over, code, text", [
    (dict(dtype=7), -2, "dtype 7"), (dict(n_tok=-1), -1, "n_tok"), (dict(n_tok=2 ** 30 + 1), -1, "n_tok"), (dict(n_seq=-2), -1, "n_seq"),
    (dict(q_heads=3), -1, "multiple of kv_heads"), (dict(kv_heads=0), -1, "multiple of kv_heads"), (dict(q_heads=0), -1, "multiple of kv_heads"),
    (dict(D=24), -1, "multiple of 16"), (dict(D=0), -1, "multiple of 16"), (dict(D=144), -2, "maximum 128"), (dict(window_size=-1), -1, "window_size"),
    (dict(row=260), -1, "multiples of 8"), (dict(head=0), -1, "multiples of 8"), (dict(row=2 ** 39), -1, "2^39"),
    (dict(dtype=2, row=512), -2, "dense"), (dict(n_tok=2 ** 30, q_heads=2 ** 10), -5, "tiles"),
])
def test_refused_shapes(capi, over, code, text):
    L = capi.lib()
    s = _shape(capi, **over)
    one = ctypes.c_void_p(4096)
    assert L.attn_b200_packed_forward(ctypes.byref(s), one, one, one, one, one, one, None) == code
    assert text in L.attn_b200_last_error().decode()
    assert L.attn_b200_packed_backward(ctypes.byref(s), *([one] * 11), None) == code


def test_refused_pointers(capi):
    L = capi.lib()
    s = _shape(capi)
    good, odd = ctypes.c_void_p(4096), ctypes.c_void_p(4104)
    for i in range(6):
        for bad, text in ((None, "null"), (odd, "aligned")):
            args = [good] * 6
            args[i] = bad
            if i == 5 and bad is odd:
                continue      # L is read by elements
            assert L.attn_b200_packed_forward(ctypes.byref(s), *args, None) == -1
            assert text in L.attn_b200_last_error().decode()
    assert L.attn_b200_packed_forward(None, *([good] * 6), None) == -1
    assert L.attn_b200_packed_plan(None, 4, 1, good, None) == -1
    assert L.attn_b200_packed_plan(good, 4, 1, odd, None) == -1
    assert L.attn_b200_packed_plan(good, -4, 1, good, None) == -1
    assert L.attn_b200_packed_plan_ints(-1, 2) == 0
    assert L.attn_b200_packed_plan_ints(0, 0) == 8 + 8 * 2 + 4 * 2
    assert L.attn_b200_packed_plan_ints(1000, 3) == 8 + 8 * (1000 // 128 + 3 + 2) + 4 * (1000 // 256 + 3 + 2) + 2 * 3


def test_empty_batch_needs_no_device(capi):
    L = capi.lib()
    s = _shape(capi, n_tok=0)
    assert L.attn_b200_packed_forward(ctypes.byref(s), *([None] * 6), None) == 0
    assert L.attn_b200_packed_backward(ctypes.byref(s), *([None] * 11), None) == 0
    assert L.attn_b200_packed_backward_scratch_bytes(ctypes.byref(_shape(capi))) == 4 * 256 * 4


def test_python_refusals(packed):
    cpu = torch.zeros(3, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="CUDA tensor"):
        packed.packed_plan(cpu, 4)
    with pytest.raises(ValueError, match="max_seqlen"):
        packed.packed_plan(cpu, 4, max_seqlen=-1)
    plan = packed.PackedPlan(torch.zeros(50, dtype=torch.int32), 4, 2, None)
    x = torch.zeros(4, 2, 16)
    with pytest.raises(RuntimeError, match="CUDA tensors"):
        packed.packed_attention(x, x, x, plan)


# ---- plain implementation in 64 bits, with bounds ----------------------------------------------------

def reference(q, k, v, do, cu, window):
    """(O, dq, dk, dv) and a bound of the error of each.  u: half a step of the type that P and dS are rounded to
    (0 in fp32) and results are stored in.  A score is a sum of D products, off by at most (D + 4) 2^-24 of the sum
    of their sizes, so is P relatively by the largest such error of its row, twice (the normaliser has one too); sums
    of n products in fp32 are off by n 2^-24 of the sum of their sizes.  eta: P and dS below the type's normal numbers (6e-5 in
    fp16) are off by up to half of its smallest step, 2^-25, whatever their size; in the forward P is rounded in units of
    a row's largest or smaller, so that its eta is no larger."""
    dt = q.dtype
    u = 0.0 if dt == torch.float32 else torch.finfo(dt).eps / 2
    out_u = torch.finfo(dt).eps / 2
    f = 2.0 ** -24
    tiny = torch.finfo(dt).smallest_normal * torch.finfo(dt).eps
    eta = 0.0 if dt == torch.float32 else tiny / 2
    n_tok, H, D = q.shape
    Hkv, group, s = k.shape[1], H // k.shape[1], 1 / math.sqrt(D)
    q, k, v, do = (t.double() for t in (q, k, v, do))
    res = [torch.zeros_like(t) for t in (q, q, k, v)]
    err = [torch.zeros_like(t) for t in (q, q, k, v)]
    for a, b in zip(cu[:-1], cu[1:]):
        n = b - a
        if n == 0:
            continue
        i = torch.arange(n, device=q.device)
        seen = (i[None] <= i[:, None]) & (i[:, None] < i[None] + (window if window is not None else n))
        for h in range(H):
            qh, kh, vh, gh = q[a:b, h], k[a:b, h // group], v[a:b, h // group], do[a:b, h]
            S = (qh @ kh.T * s).masked_fill(~seen, -math.inf)
            P = torch.softmax(S, -1).nan_to_num(0.0)
            size = (qh.abs() @ kh.abs().T * s * (D + 4) * f).masked_fill(~seen, 0.0)
            rel = u + 2 * size.amax(-1, keepdim=True) + (n + 16) * f            # of P
            acc = (n * group + 16) * f                                          # of a sum of up to n group products
            O = P @ vh
            eO = (rel * P + eta * seen) @ vh.abs() + acc * (P @ vh.abs()) + out_u * O.abs()
            dP = gh @ vh.T
            eP = (gh.abs() @ vh.abs().T) * (D + 4) * f
            Dv = (P * dP).sum(-1, keepdim=True)
            eD = (gh.abs() * (eO + out_u * O.abs())).sum(-1, keepdim=True) + (gh.abs() * O.abs()).sum(-1, keepdim=True) * (D + 4) * f
            dS = P * (dP - Dv)
            eS = (rel + u + 4 * f) * dS.abs() + P * (eP + eD) * (1 + u) + eta * seen
            res[0][a:b, h] = O
            err[0][a:b, h] = eO
            res[1][a:b, h] = dS @ kh * s
            err[1][a:b, h] = (eS + acc * dS.abs()) @ kh.abs() * s
            res[2][a:b, h // group] += dS.T @ qh * s
            err[2][a:b, h // group] += (eS + acc * dS.abs()).T @ qh.abs() * s
            res[3][a:b, h // group] += P.T @ gh
            err[3][a:b, h // group] += ((rel + acc) * P + eta * seen).T @ gh.abs()
    for i in (1, 2, 3):
        err[i] += out_u * res[i].abs()
    # results below the type's normal numbers are off by half of its smallest step; second-order terms: 2 %
    return res, [e * 1.02 + tiny for e in err]


def tensors(n_tok, H, Hkv, D, dtype, seed=0, amp=1.0):
    g = torch.Generator().manual_seed(seed)
    r = lambda h, a=1.0: (torch.randn(n_tok, h, D, generator=g) * a).to(dtype).cuda()
    return r(H, amp), r(Hkv, amp), r(Hkv), r(H)


def both_passes(packed, q, k, v, do, plan, window):
    q, k, v = (t.detach().requires_grad_(True) for t in (q, k, v))
    o = packed.packed_attention(q, k, v, plan, window)
    return [o.detach(), *torch.autograd.grad(o, (q, k, v), do)]


def check(packed, lens, H, Hkv, D, dtype, window=None, front=0, tail=0, amp=1.0, seed=0):
    cu = offsets(lens, front)
    n_tok = cu[-1] + tail
    q, k, v, do = tensors(n_tok, H, Hkv, D, dtype, seed, amp)
    plan = packed.packed_plan(torch.tensor(cu, dtype=torch.int32, device="cuda"), n_tok)
    got = both_passes(packed, q, k, v, do, plan, window)
    want, bound = reference(q, k, v, do, cu, window)
    for name, x, w, b in zip(("O", "dq", "dk", "dv"), got, want, bound):
        assert x.dtype == dtype and x.shape == w.shape and x.is_contiguous()
        worst = ((x.double() - w).abs() / b).max() if x.numel() else torch.tensor(0.0)
        assert bool(worst <= 1), (name, float(worst))
    if n_tok:
        no_graph = packed.packed_attention(q, k, v, plan, window)
        assert torch.equal(no_graph, got[0])


RAGGED = [1, 63, 64, 0, 65, 127, 128, 129, 300]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("H, Hkv, D", [(2, 2, 64), (4, 1, 128), (6, 2, 80), (3, 3, 16), (2, 1, 112), (4, 2, 32)])
def test_ragged_lengths(packed, dtype, H, Hkv, D):
    check(packed, RAGGED, H, Hkv, D, dtype, tail=5, front=3)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("window", [0, 1, 17, 64, 100, 129, 2 ** 31, 2 ** 40])
@pytest.mark.parametrize("D", [64, 128])
def test_windows(packed, dtype, window, D):
    check(packed, [1, 40, 130, 0, 333], 4, 2, D, dtype, window=window, tail=2)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("lens, tail", [([1], 0), ([0], 0), ([0, 0], 7), ([], 130), ([2], 0), ([1] * 9, 0), ([700], 0)])
def test_few_rows(packed, dtype, lens, tail):
    check(packed, lens, 2, 1, 64, dtype, tail=tail)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype, D", [(torch.bfloat16, 64), (torch.float16, 128)])
def test_many_tiles(packed, dtype, D):
    # two CTAs per SM in the forward (both passes at D = 64), more CTAs than fit at a time
    check(packed, [517, 1, 1200, 90, 64, 64, 3, 260, 31], 24, 8, D, dtype, tail=9)


# long sequences, for which the forward takes its query tiles in pairs: mean lengths from 1024 (D <= 64) and 4096 on, 185 pairs and more
PAIRS = [([1500, 700, 2300, 1], 24, 12, 64), ([1100, 1281], 32, 4, 32), ([4200], 16, 4, 128), ([129, 8100], 12, 4, 80)]


@pytest.mark.gpu
@pytest.mark.parametrize("lens, H, Hkv, D", PAIRS)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_long_sequences(packed, lens, H, Hkv, D, dtype):
    check(packed, lens, H, Hkv, D, dtype, front=3, tail=1)


@pytest.mark.gpu
@pytest.mark.parametrize("window", [0, 1, 2, 100, 127, 128, 129, 256, 300, 1000])
@pytest.mark.parametrize("lens, H, Hkv, D", PAIRS[:1] + PAIRS[2:3])
def test_long_sequences_with_windows(packed, lens, H, Hkv, D, window):
    check(packed, lens, H, Hkv, D, torch.bfloat16, window=window, tail=300)


@pytest.mark.gpu
@pytest.mark.parametrize("n", [1025, 1152, 1153, 1279, 1280, 1281, 1407, 1408, 1409])
def test_last_rows_of_a_pair(packed, n):
    check(packed, [n, n], 24, 8, 64, torch.bfloat16, amp=3.0)


@pytest.mark.gpu
@pytest.mark.parametrize("lens, D, dtype", [([1300, 900, 1200], 64, torch.bfloat16), ([4100, 4300], 128, torch.float16)])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_long_sequences_do_not_touch_one_another(packed, lens, D, dtype, bad):
    cu = offsets(lens, 5)
    n_tok = cu[-1] + 9
    q, k, v, _ = tensors(n_tok, 24, 4, D, dtype)
    plan = packed.packed_plan(torch.tensor(cu, dtype=torch.int32, device="cuda"), n_tok)
    clean = packed.packed_attention(q, k, v, plan)
    for t in (q, k, v):
        for a, b in ((0, 5), (cu[1], cu[2]), (cu[-1], n_tok)):
            t[a:b] = bad
    dirty = packed.packed_attention(q, k, v, plan)
    for i in range(len(lens)):
        a, b = cu[i], cu[i + 1]
        assert torch.equal(clean[a:b], dirty[a:b]) if i != 1 else bool(dirty[a:b].isnan().all()) or bad == -math.inf
    assert not bool(dirty[:5].any()) and not bool(dirty[cu[-1]:].any())
    # a key that is not a number reaches the rows that see it
    q, k, v, _ = tensors(n_tok, 24, 4, D, dtype)
    at = cu[0] + 700
    k[at] = math.nan
    o = packed.packed_attention(q, k, v, plan)
    assert bool(o[at:cu[1]].isnan().all()) and not bool(o[:at].isnan().any()) and not bool(o[cu[1]:].isnan().any())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_peaked_rows(packed, dtype):
    check(packed, [200, 77, 350], 4, 2, 64, dtype, amp=4.0)


@pytest.mark.gpu
def test_a_thousand_short_sequences(packed):
    lens = [(7 * i) % 23 for i in range(1500)]      # more than a pass of the plan takes at a time
    check(packed, lens, 2, 1, 32, torch.bfloat16, front=1, tail=1)


def gaps_of(cu, n_tok, step):
    first, last = (min(max(c, 0), n_tok) for c in (cu[0], max(cu)))
    return [(r, -1, first) for r in range(0, first, step)] + [(r, -1, n_tok) for r in range(last, n_tok, step)]


def plain_plan(cu, n_tok):
    """(tiles of queries, tiles of keys) as (row0, begin, end) -> length of the stream in tiles; rows of no sequence"""
    fixed, top = [], 0
    for c in cu:
        top = max(top, min(max(c, 0), n_tok))
        fixed.append(top)
    rows, cols = {}, {}
    for a, b in zip(fixed[:-1], fixed[1:]):
        n = (b - a + 127) // 128
        for t in range(n):
            rows[(a + 128 * t, a, b)] = t + 1
            cols[(a + 128 * t, a, b)] = n - t
    return rows, cols, gaps_of(cu, n_tok, 128), max([b - a for a, b in zip(fixed[:-1], fixed[1:])], default=0)


@pytest.mark.gpu
@pytest.mark.parametrize("cu, n_tok", [
    ([0, 5, 5, 300, 1000], 1000), ([0], 0), ([0], 300), ([4, 200], 900), ([0, 700, 300, 800], 900), ([-5, 10, 2000], 129),
    (offsets([(37 * i) % 301 for i in range(2500)]), 400000), ([0, 300000], 300001), ([0, 128], 128),
])
@pytest.mark.parametrize("dtype", [torch.int32, torch.int64])
def test_plan(packed, cu, n_tok, dtype):
    plan = packed.packed_plan(torch.tensor(cu, dtype=dtype, device="cuda"), n_tok)
    t = plan.tensor.cpu()
    cap = n_tok // 128 + len(cu) - 1 + 2
    rows, cols, gaps, longest = plain_plan(cu, n_tok)
    assert int(t[0]) == len(rows) and int(t[1]) == longest
    for first, want in ((8, rows), (8 + 4 * cap, cols)):
        e = [tuple(x[:3]) for x in t[first:first + 4 * cap].view(cap, 4).tolist()]
        n = len(rows)
        assert sorted(e[:n]) == sorted(want) and e[n:n + len(gaps)] == gaps and all(x[0] == -1 for x in e[n + len(gaps):])
        work = [want[x] for x in e[:n]]
        shift = 0                              # long streams share one of 2047 bins
        while (n_tok // 128 >> shift) >= 2047:
            shift += 1
        bins = [(x - 1) >> shift for x in work]
        assert bins == sorted(bins, reverse=True)      # longest streams first
    pair_cap = n_tok // 256 + len(cu) - 1 + 2
    e = [tuple(x[:3]) for x in t[8 + 8 * cap:8 + 8 * cap + 4 * pair_cap].view(pair_cap, 4).tolist()]
    want = {k: v for k, v in rows.items() if (k[0] - k[1]) % 256 == 0}
    n, wide_gaps = len(want), gaps_of(cu, n_tok, 256)
    assert sorted(e[:n]) == sorted(want) and e[n:n + len(wide_gaps)] == wide_gaps and all(x[0] == -1 for x in e[n + len(wide_gaps):])
    bins = [(want[x] - 1) >> shift for x in e[:n]]
    assert bins == sorted(bins, reverse=True)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype, D", [(torch.bfloat16, 64), (torch.float16, 128), (torch.float32, 80)])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_sequences_do_not_touch_one_another(packed, dtype, D, bad):
    lens, H, Hkv = [70, 200, 33, 129], 4, 2
    cu = offsets(lens, 6)
    n_tok = cu[-1] + 50
    q, k, v, do = tensors(n_tok, H, Hkv, D, dtype)
    plan = packed.packed_plan(torch.tensor(cu, dtype=torch.int32, device="cuda"), n_tok)
    clean = both_passes(packed, q, k, v, do, plan, None)
    for t in (q, k, v, do):
        for a, b in ((0, 6), (cu[1], cu[2]), (cu[3], n_tok)):      # in front, the second and the last sequence, behind
            t[a:b] = bad
    dirty = both_passes(packed, q, k, v, do, plan, None)
    for a, b in ((0, 6), (cu[0], cu[1]), (cu[2], cu[3]), (cu[-1], n_tok)):
        for x, y in zip(clean, dirty):
            assert torch.equal(x[a:b], y[a:b])
    assert bool(dirty[0][cu[1]:cu[2]].isnan().all()) if bad != -math.inf else True
    # a sequence by itself gives the same as within the batch, but for the order of its sums where few tiles are shared among CTAs
    eps = torch.finfo(dtype).eps
    for i in (0, 2):
        a, b = cu[i], cu[i + 1]
        alone = packed.packed_plan(torch.tensor([0, b - a], dtype=torch.int32, device="cuda"), b - a)
        for x, y in zip(clean, both_passes(packed, *(t[a:b].contiguous() for t in (q, k, v, do)), alone, None)):
            assert bool(((x[a:b] - y).abs().float() <= 2 * eps * y.abs().float() + 300 * 2.0 ** -24 * float(y.abs().max())).all())


@pytest.mark.gpu
def test_nan_in_a_visible_key_is_seen(packed):
    for dtype in (torch.bfloat16, torch.float32):
        q, k, v, _ = tensors(300, 2, 2, 64, dtype)
        k[130] = math.nan
        plan = packed.packed_plan(torch.tensor([0, 300], dtype=torch.int32, device="cuda"), 300)
        o = packed.packed_attention(q, k, v, plan)
        assert bool(o[130:].isnan().all()) and not bool(o[:130].isnan().any())


@pytest.mark.gpu
def test_offsets_out_of_order_are_cut(packed):
    q, k, v, do = tensors(500, 2, 1, 64, torch.bfloat16)
    cu = torch.tensor([-3, 200, 90, 1 << 30, 7], dtype=torch.int32, device="cuda")
    same = torch.tensor([0, 200, 200, 500, 500], dtype=torch.int32, device="cuda")
    for x, y in zip(both_passes(packed, q, k, v, do, packed.packed_plan(cu, 500), None), both_passes(packed, q, k, v, do, packed.packed_plan(same, 500), None)):
        assert torch.equal(x, y)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_strides(packed, dtype):
    n, H, Hkv, D = 333, 4, 2, 64
    cu = torch.tensor([0, 100, 333], dtype=torch.int32, device="cuda")
    plan = packed.packed_plan(cu, n)
    g = torch.Generator().manual_seed(3)
    qkv = torch.randn(n, H + 2 * Hkv, D, generator=g).to(dtype).cuda()
    heads_first = torch.randn(H, n, D, generator=g).to(dtype).cuda()
    odd = torch.randn(n, Hkv, D + 1, generator=g).to(dtype).cuda()
    shifted = torch.randn(n * Hkv * D + 1, generator=g).to(dtype).cuda()[1:].view(n, Hkv, D)
    do = torch.randn(n, H, 2 * D, generator=g).to(dtype).cuda()[:, :, ::2]
    one = torch.randn(n, 1, D, generator=g).to(dtype).cuda().expand(n, Hkv, D)
    views = [(qkv[:, :H], qkv[:, H:H + Hkv], qkv[:, H + Hkv:]), (heads_first.transpose(0, 1), odd[:, :, 1:], shifted), (qkv[:, :H], one, odd[:, :, :D])]
    for q, k, v in views:
        got = both_passes(packed, q, k, v, do, plan, None)
        want = both_passes(packed, q.contiguous(), k.contiguous(), v.contiguous(), do.contiguous(), plan, None)
        for x, y in zip(got, want):
            assert torch.equal(x, y)
    # the gradient of a broadcast head is the sum over its uses, of one projection's result one tensor
    leaf = torch.randn(n, 1, D, generator=g).to(dtype).cuda().requires_grad_(True)
    o = packed.packed_attention(qkv[:, :H], leaf.expand(n, Hkv, D), qkv[:, H + Hkv:], plan)
    (gl,) = torch.autograd.grad(o, leaf, do)
    dk = both_passes(packed, qkv[:, :H], leaf.detach().expand(n, Hkv, D), qkv[:, H + Hkv:], do, plan, None)[2]
    assert gl.shape == leaf.shape and torch.allclose(gl.float(), dk.float().sum(1, keepdim=True), rtol=torch.finfo(dtype).eps, atol=1e-6)


@pytest.mark.gpu
def test_refused_calls_on_the_device(packed):
    q, k, v, _ = tensors(64, 4, 2, 64, torch.bfloat16)
    plan = packed.packed_plan(torch.tensor([0, 64], dtype=torch.int32, device="cuda"), 64)
    ok = packed.packed_attention
    for args, text in (((q[:, :3], k, v), "multiple"), ((q, k, v[:, :1]), "same shape"), ((q.half(), k, v), "same dtype"), ((q, k[:32], v[:32]), "agree"),
                       ((q[:32], k[:32], v[:32]), "plan"), ((q[0], k, v), "n_tok, heads"), ((q.double(), k.double(), v.double()), "fp16, bf16 or fp32"),
                       ((q[..., :24], k[..., :24], v[..., :24]), "multiple of 16"), ((q.cpu(), k, v), "CUDA")):
        with pytest.raises(RuntimeError, match=text):
            ok(*args, plan)
    with pytest.raises(RuntimeError, match="window_size"):
        ok(q, k, v, plan, -1)
    with pytest.raises(RuntimeError, match="int32 or int64"):
        packed.packed_plan(torch.zeros(2, device="cuda"), 4)
    with pytest.raises(RuntimeError, match="n_tok"):
        packed.packed_plan(torch.zeros(2, dtype=torch.int32, device="cuda"), -1)
    with pytest.raises(RuntimeError, match="traced"):
        torch.jit.trace(lambda x: ok(x, k, v, plan), (q,))
    import torch.autograd.forward_ad as fad
    with fad.dual_level(), pytest.raises(RuntimeError, match="forward-mode"):
        ok(fad.make_dual(q, q), k, v, plan)
    with pytest.raises(RuntimeError):
        torch.func.grad(lambda x: ok(x, k, v, plan).float().sum())(q)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("H, Hkv, D", [(6, 2, 64), (4, 4, 128), (5, 1, 80)])
def test_one_visible_key_takes_no_gradient_of_scores(packed, dtype, H, Hkv, D):
    # P = 1 whatever the score is: dq and dk are 0, not nearly
    for lens, window in (([1], None), ([1, 1, 0, 1], None), ([70, 1, 200], 1)):
        cu = offsets(lens)
        q, k, v, do = tensors(cu[-1] + 2, H, Hkv, D, dtype)
        plan = packed.packed_plan(torch.tensor(cu, dtype=torch.int32, device="cuda"), cu[-1] + 2)
        o, dq, dk, dv = both_passes(packed, q, k, v, do, plan, window)
        assert not bool(dq.any()) and not bool(dk.any()) and bool(dv[:cu[-1]].flatten(1).any(1).all())
        assert torch.equal(o[:cu[-1]], v[:cu[-1]].repeat_interleave(H // Hkv, 1))
    # the first row of a sequence, beside rows that see more; a score that is not a number stays one
    cu = [0, 130, 137, 400]
    q, k, v, do = tensors(400, H, Hkv, D, dtype)
    plan = packed.packed_plan(torch.tensor(cu, dtype=torch.int32, device="cuda"), 400)
    dq = both_passes(packed, q, k, v, do, plan, None)[1]
    assert (dq == 0).flatten(1).all(1).nonzero().flatten().tolist() == cu[:-1]
    do[:] = 0
    do[130] = 1
    assert not any(bool(t.any()) for t in both_passes(packed, q, k, v, do, plan, None)[1:3])
    q[130, 0, 3] = math.nan
    o, dq, dk, dv = both_passes(packed, q, k, v, do, plan, None)
    assert bool(o[130, 0].isnan().all()) and bool(dq[130, 0].isnan().all()) and bool(dk[130, 0].isnan().any())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("H, Hkv, D", [(6, 2, 32), (4, 4, 128), (5, 1, 80)])
@pytest.mark.parametrize("window", [None, 3])
def test_gradients_of_sequences_of_few_rows(packed, dtype, H, Hkv, D, window):
    # D without the rounding of O: what is left is dS and the result, rounded once each (u = half a step), and P, dP and D in float, relatively
    # within 2^-16 for D + 8 terms of scores below 16.  In fp16 dS is also off by half of its smallest step, 2^-25
    lens = [7, 2, 0, 8, 5, 1, 3, 4, 6]
    cu, u, s = offsets(lens, 2), torch.finfo(dtype).eps / 2, 1 / math.sqrt(D)
    q, k, v, do = tensors(cu[-1] + 3, H, Hkv, D, dtype, seed=2, amp=1.4)
    plan = packed.packed_plan(torch.tensor(cu, dtype=torch.int32, device="cuda"), cu[-1] + 3)
    got = both_passes(packed, q, k, v, do, plan, window)[1:3]
    eta = torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
    want, err = [torch.zeros_like(t, dtype=torch.float64) for t in (q, k)], [torch.zeros_like(t, dtype=torch.float64) for t in (q, k)]
    for a, b in zip(cu[:-1], cu[1:]):
        i = torch.arange(b - a, device="cuda")
        seen = (i[None] <= i[:, None]) & (i[:, None] < i[None] + (window or b - a))
        for h in range(H if b > a else 0):
            qh, kh, vh, gh = (t[a:b, x].double() for t, x in ((q, h), (k, h * Hkv // H), (v, h * Hkv // H), (do, h)))
            P = torch.softmax((qh @ kh.T * s).masked_fill(~seen, -math.inf), -1)
            dP = gh @ vh.T
            dS = P * (dP - (P * dP).sum(-1, keepdim=True))
            size = P * (gh.abs() @ vh.abs().T + (P * (gh.abs() @ vh.abs().T)).sum(-1, keepdim=True))
            eS = (u * dS.abs() + 2.0 ** -16 * size) * 1.01 + eta * seen
            want[0][a:b, h] = dS @ kh * s
            want[1][a:b, h * Hkv // H] += dS.T @ qh * s
            err[0][a:b, h] = eS @ kh.abs() * s
            err[1][a:b, h * Hkv // H] += eS.T @ qh.abs() * s
    for x, w, e in zip(got, want, err):
        worst = ((x.double() - w).abs() / (e + 1.01 * u * w.abs() + eta)).max()
        assert bool(worst <= 1), float(worst)


@pytest.mark.gpu
def test_captured_plan_and_passes(packed):
    n, H, Hkv, D = 700, 4, 2, 64
    q, k, v, do = tensors(n, H, Hkv, D, torch.bfloat16)
    cu = torch.tensor([0, 200, 640], dtype=torch.int32, device="cuda")

    def step():
        return both_passes(packed, q, k, v, do, packed.packed_plan(cu, n), 300)
    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for lens in ([0, 200, 640], [0, 0, 700], [10, 500, 501], [0, 333, 650]):
        cu.copy_(torch.tensor(lens, dtype=torch.int32))
        for t in (q, k, v, do):
            t.copy_(torch.randn(t.shape))
        graph.replay()
        for x, y in zip(out, step()):
            assert torch.equal(x, y)


@pytest.mark.gpu
@pytest.mark.parametrize("H, Hkv, D", [(16, 16, 64), (32, 8, 128)])
def test_captured_long_sequences(packed, H, Hkv, D):
    # forwards of pairs of tiles; lengths of another replay
    n = 8300
    q, k, v, do = tensors(n, H, Hkv, D, torch.bfloat16)
    cu = torch.tensor([0, 8200], dtype=torch.int32, device="cuda")

    def step():
        return both_passes(packed, q, k, v, do, packed.packed_plan(cu, n), None)
    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for lens in ([0, 8200], [5, 8300], [0, 1]):
        cu.copy_(torch.tensor(lens, dtype=torch.int32))
        graph.replay()
        for x, y in zip(out, step()):
            assert torch.equal(x, y)


@pytest.mark.gpu
def test_captured_second_derivative(packed):
    # with the length of the longest sequence given, nothing waits for the host
    n, H, Hkv, D = 260, 4, 2, 64
    leaves = [t.requires_grad_(True) for t in tensors(n, H, Hkv, D, torch.bfloat16)]
    tangents = tensors(n, H, Hkv, D, torch.bfloat16, seed=3)[:3]
    cu = torch.tensor([0, 100, 256], dtype=torch.int32, device="cuda")

    def step(leaves):
        first = torch.autograd.grad(packed.packed_attention(*leaves[:3], packed.packed_plan(cu, n, max_seqlen=200)), leaves[:3], leaves[3], create_graph=True)
        return torch.autograd.grad(first, leaves, tangents)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step(leaves)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            out = step(leaves)
    for lens in ([0, 100, 256], [3, 200, 260], [0, 0, 190]):
        cu.copy_(torch.tensor(lens, dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        for x, y in zip(out, step([t.detach().requires_grad_(True) for t in leaves])):
            assert torch.equal(x, y)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_some_gradients_and_their_layouts(packed, dtype):
    q, k, v, do = tensors(300, 4, 2, 64, dtype)
    plan = packed.packed_plan(torch.tensor([0, 130, 290], dtype=torch.int64, device="cuda"), 300)
    want = both_passes(packed, q, k, v, torch.ones_like(do), plan, None)
    # the gradient of a sum has strides of 0; each input alone; the same graph twice
    for i in range(3):
        leaves = [t.detach().clone() for t in (q, k, v)]
        leaves[i].requires_grad_(True)
        o = packed.packed_attention(*leaves, plan)
        for _ in range(2):
            assert torch.equal(torch.autograd.grad(o.sum(), leaves[i], retain_graph=True)[0], want[1 + i])
    # a gradient laid out by heads
    leaves = [t.detach().clone().requires_grad_(True) for t in (q, k, v)]
    o = packed.packed_attention(*leaves, plan)
    by_heads = do.transpose(0, 1).contiguous().transpose(0, 1)
    for a, b in zip(torch.autograd.grad(o, leaves, by_heads), both_passes(packed, q, k, v, do, plan, None)[1:]):
        assert torch.equal(a, b)
    # one tensor in all three places
    x = k.detach().clone().requires_grad_(True)
    got = torch.autograd.grad(packed.packed_attention(x, x, x, plan), x, do[:, :2])[0]
    parts = both_passes(packed, k, k, k, do[:, :2], plan, None)[1:]
    assert float((got.float() - sum(t.float() for t in parts)).norm() / got.float().norm()) <= 2 * torch.finfo(dtype).eps


@pytest.mark.gpu
def test_second_derivative_without_rows_or_keys(packed):
    for n, cu, window, longest in ((0, [0], None, None), (5, [0], None, None), (5, [0, 0, 0], None, None), (70, [0, 70], 0, None), (70, [0, 70], None, 0)):
        leaves = [t.requires_grad_(True) for t in tensors(n, 4, 2, 32, torch.bfloat16)]
        plan = packed.packed_plan(torch.tensor(cu, dtype=torch.int32, device="cuda"), n, max_seqlen=longest)
        first = torch.autograd.grad(packed.packed_attention(*leaves[:3], plan, window), leaves[:3], leaves[3], create_graph=True)
        for t, x in zip(torch.autograd.grad(first, leaves, [torch.ones_like(f) for f in first]), leaves):
            assert t.shape == x.shape and not bool(t.any())


@pytest.mark.gpu
@pytest.mark.parametrize("n, H, Hkv, D, dtype, window, bad", [
    (300, 4, 2, 64, torch.bfloat16, 150, 120), (300, 4, 2, 128, torch.bfloat16, 150, 120), (300, 4, 2, 64, torch.float32, 150, 120),
    (4100, 16, 16, 64, torch.bfloat16, 1500, 1100), (8200, 16, 4, 128, torch.bfloat16, 1500, 1100)])
def test_scores_of_minus_infinity_count_nothing(packed, n, H, Hkv, D, dtype, window, bad):
    # keys 1 .. bad: products below the range of float, as beside them finite ones of -1e4 with probabilities of 0 too.  Every row
    # sees another key, with the window some behind whole tiles of these
    q, k, v, do = tensors(n, H, Hkv, D, dtype)
    q, k = torch.full_like(q, 2.0 ** 64), k * 2.0 ** -64
    plan = packed.packed_plan(torch.tensor([0, n], dtype=torch.int32, device="cuda"), n)
    out = []
    for low in (-2.0 ** 66, -1250 * 2.0 ** -64):
        k[1:bad + 1] = low
        out.append(both_passes(packed, q, k, v, do, plan, window))
    for a, b in zip(*out):
        assert bool(a.isfinite().all()) and torch.equal(a, b)


@pytest.mark.gpu
def test_two_streams_at_once(packed):
    cases = []
    for seed, lens in ((1, [300, 400]), (2, [650, 50])):
        q, k, v, do = tensors(700, 8, 2, 128, torch.bfloat16, seed)
        plan = packed.packed_plan(torch.tensor(offsets(lens), dtype=torch.int32, device="cuda"), 700)
        cases.append(((q, k, v, do, plan, None), both_passes(packed, q, k, v, do, plan, None)))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    for _ in range(5):
        got = []
        for st, (args, _) in zip(streams, cases):
            with torch.cuda.stream(st):
                got.append(both_passes(packed, *args))
        torch.cuda.synchronize()
        for g, (_, want) in zip(got, cases):
            assert all(torch.equal(x, y) for x, y in zip(g, want))


def _math_attention(q, k, v, cu, window):
    out = []
    for a, b in zip(cu[:-1], cu[1:]):
        i = torch.arange(b - a)
        seen = (i[None] <= i[:, None]) & (i[:, None] < i[None] + (window or b - a))
        kk, vv = (t[a:b].repeat_interleave(q.shape[1] // k.shape[1], 1).transpose(0, 1) for t in (k, v))
        S = (q[a:b].transpose(0, 1) @ kk.transpose(1, 2) / math.sqrt(q.shape[2])).masked_fill(~seen, -math.inf)
        out.append((torch.softmax(S, -1) @ vv).transpose(0, 1))
    return torch.cat(out)


@pytest.mark.gpu
@pytest.mark.parametrize("known", [None, 60, 64])
@pytest.mark.parametrize("dtype, tol", [(torch.float32, 2e-5), (torch.bfloat16, 3e-2)])
def test_second_derivative(packed, dtype, tol, known):
    # tol: fp32, sums of up to 60 x 4 products of sums in 2^-24 each; bf16, five rounded operands of 2^-8 each behind one
    # another and a rounded first backward, against the norm of the result
    lens, H, Hkv, D = [40, 0, 60, 1], 4, 2, 32
    cu = offsets(lens)
    n = cu[-1] + 3
    q, k, v, do = tensors(n, H, Hkv, D, dtype)
    g2 = tensors(n, H, Hkv, D, dtype, seed=9)[:3]
    plan = packed.packed_plan(torch.tensor(cu, dtype=torch.int32, device="cuda"), n, max_seqlen=known)
    leaves = [t.requires_grad_(True) for t in (q, k, v, do)]
    first = torch.autograd.grad(packed.packed_attention(q, k, v, plan, 25), (q, k, v), do, create_graph=True)
    got = torch.autograd.grad(first, leaves, g2)
    d = [t.detach().double().cpu().requires_grad_(True) for t in (q, k, v, do)]
    o = _math_attention(d[0][:cu[-1]], d[1][:cu[-1]], d[2][:cu[-1]], cu, 25)
    f64 = torch.autograd.grad(o, d[:3], d[3][:cu[-1]], create_graph=True)
    want = torch.autograd.grad(f64, d, [t.double().cpu() for t in g2])
    for x, w in zip(got, want):
        assert float((x.double().cpu() - w).norm() / w.norm()) <= tol
        assert not bool(x[cu[-1]:].any())
    with pytest.raises(RuntimeError, match="third derivative"):
        first = torch.autograd.grad(packed.packed_attention(q, k, v, plan, 25), (q, k, v), do, create_graph=True)
        torch.autograd.grad(first, leaves, g2, create_graph=True)


@pytest.mark.gpu
def test_gradient_against_differences(packed):
    # central differences of <O, do> along a direction, h = 2^-6: truncation h^2 / 6 of the third derivative, of the size of the
    # first at unit variance (4e-5), and 2 x 2^-24 x the sum's size over 2 h (under 1e-4 here); a slope is about the gradient's norm
    cu = torch.tensor([0, 90, 260], dtype=torch.int32, device="cuda")
    q, k, v, do = tensors(260, 4, 2, 64, torch.float32)
    plan = packed.packed_plan(cu, 260)
    dirs = tensors(260, 4, 2, 64, torch.float32, seed=5)[:3]
    grads = both_passes(packed, q, k, v, do, plan, 70)[1:]
    h = 2.0 ** -6
    for i in range(3):
        f = []
        for sign in (1, -1):
            args = [q, k, v]
            args[i] = args[i] + sign * h * dirs[i]
            f.append((packed.packed_attention(*args, plan, 70).double() * do.double()).sum())
        slope, want = float((f[0] - f[1]) / (2 * h)), float((grads[i].double() * dirs[i].double()).sum())
        assert abs(slope - want) <= 5e-3 * float(grads[i].double().norm())


def test_products_wait_for_their_items(tmp_path):
    # the order of the paired forward's issuing warps, walked through on the CPU
    here = os.path.dirname(os.path.abspath(__file__))
    program = str(tmp_path / "packed_order")
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Werror", "-I" + os.path.join(PKG_DIR, "csrc"), os.path.join(here, "host", "packed_order.cpp"), "-o", program], check=True)
    done = subprocess.run([program], capture_output=True, text=True, timeout=120)
    assert done.returncode == 0, done.stdout + done.stderr


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("H, Hkv, D", [(6, 2, 32), (4, 4, 128), (5, 1, 80), (2, 1, 64)])
@pytest.mark.parametrize("window", [2, 3, 5, 7, 8])
def test_gradients_under_narrow_windows(packed, dtype, H, Hkv, D, window):
    # every row sees few keys, whichever place it has in its sequence: the bound of test_gradients_of_sequences_of_few_rows, D without the rounding of O
    lens = [300, 5, 0, 128, 129, 16, 1, 17]
    cu, u, s, f = offsets(lens, 3), torch.finfo(dtype).eps / 2, 1 / math.sqrt(D), 2.0 ** -16
    n = cu[-1] + 40
    q, k, v, do = tensors(n, H, Hkv, D, dtype, seed=4, amp=1.4)
    plan = packed.packed_plan(torch.tensor(cu, dtype=torch.int32, device="cuda"), n)
    got = both_passes(packed, q, k, v, do, plan, window)[1:3]
    eta = torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
    at = torch.arange(n, device="cuda")
    seq = torch.bucketize(at, torch.tensor(cu, device="cuda"), right=True)
    seen = (seq[None] == seq[:, None]) & (at[None] <= at[:, None]) & (at[:, None] < at[None] + window) & (at >= cu[0]) & (at < cu[-1])
    q, k, v, do = (t.double().transpose(0, 1) for t in (q, k.repeat_interleave(H // Hkv, 1), v.repeat_interleave(H // Hkv, 1), do))
    P = torch.softmax((q @ k.transpose(1, 2) * s).masked_fill(~seen, -math.inf), -1).nan_to_num(0.0)
    dP, size = do @ v.transpose(1, 2), do.abs() @ v.abs().transpose(1, 2)
    dS = P * (dP - (P * dP).sum(-1, keepdim=True))
    eS = (u * dS.abs() + f * P * (size + (P * size).sum(-1, keepdim=True))) * 1.01 + eta * seen
    group = lambda t: t.view(Hkv, H // Hkv, n, D).sum(1)
    for x, w, e in zip(got, (dS @ k * s, group(dS.transpose(1, 2) @ q * s)), (eS @ k.abs() * s, group(eS.transpose(1, 2) @ q.abs() * s))):
        worst = ((x.double().transpose(0, 1) - w).abs() / (e + 1.01 * u * w.abs() + eta)).max()
        assert bool(worst <= 1), float(worst)


def second_derivatives(packed, leaves, cu, n, window, tangents, known):
    plan = packed.packed_plan(torch.tensor(cu, dtype=torch.int32, device="cuda"), n, max_seqlen=known)
    leaves = [t.detach().requires_grad_(True) for t in leaves]
    first = torch.autograd.grad(packed.packed_attention(*leaves[:3], plan, window), leaves[:3], leaves[3], create_graph=True)
    return torch.autograd.grad(first, leaves, tangents)


@pytest.mark.gpu
@pytest.mark.parametrize("known", [None, 700, 800])
@pytest.mark.parametrize("dtype, tol", [(torch.float32, 2e-5), (torch.bfloat16, 3e-2)])
@pytest.mark.parametrize("window", [None, 25])
def test_second_derivative_of_unlike_lengths(packed, dtype, tol, known, window):
    # a long sequence beside short and empty ones, several calls of the dense kernels: the tolerances of test_second_derivative
    lens, H, Hkv, D = [3, 0, 11, 700, 1, 90, 0, 60, 200, 7, 7, 7], 4, 2, 32
    cu = offsets(lens, 2)
    n = cu[-1] + 3
    leaves, g2 = tensors(n, H, Hkv, D, dtype), tensors(n, H, Hkv, D, dtype, seed=9)[:3]
    got = second_derivatives(packed, leaves, cu, n, window, g2, known)
    d = [t.double().cpu().requires_grad_(True) for t in leaves]
    o = _math_attention(*d[:3], cu, window)
    want = torch.autograd.grad(torch.autograd.grad(o, d[:3], d[3][2:cu[-1]], create_graph=True), d, [t.double().cpu() for t in g2])
    for x, w in zip(got, want):
        assert float((x.double().cpu() - w).norm() / w.norm()) <= tol
        assert not bool(x[:2].any()) and not bool(x[cu[-1]:].any())


@pytest.mark.gpu
@pytest.mark.parametrize("known", [None, 2048])
def test_second_derivative_takes_memory_by_rows(packed, known):
    # one document beside 600 short ones: no more than 40 tensors of twice the batch's rows or of 128 MB, where rows padded to the longest one take 1.2 GB each
    # (15.4 GB in all)
    lens, H, D = [5] * 300 + [2048] + [11] * 300, 8, 64
    cu = offsets(lens)
    leaves, g2 = tensors(cu[-1], H, H, D, torch.bfloat16), tensors(cu[-1], H, H, D, torch.bfloat16, seed=9)[:3]
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    second_derivatives(packed, leaves, cu, cu[-1], None, g2, known)
    assert torch.cuda.max_memory_allocated() - before <= 40 * max(2 * leaves[0].numel() * 2, 128 << 20)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_second_derivative_of_a_longer_sequence_than_given_is_not_a_number(packed, dtype):
    cu, n = [0, 40, 110, 111], 115
    leaves, g2 = tensors(n, 4, 2, 32, dtype), tensors(n, 4, 2, 32, dtype, seed=9)[:3]
    for known in (1, 40, 69):
        assert all(bool(t.isnan().all()) for t in second_derivatives(packed, leaves, cu, n, None, g2, known))
    want = second_derivatives(packed, leaves, cu, n, None, g2, None)
    for known in (70, 114, 115, 2 ** 40):
        for a, b in zip(second_derivatives(packed, leaves, cu, n, None, g2, known), want):
            assert bool(a.isfinite().all()) and float((a.float() - b.float()).norm() / b.float().norm()) <= 4 * torch.finfo(dtype).eps


@pytest.mark.gpu
@pytest.mark.parametrize("known", [None, 100])
def test_second_derivative_of_no_plan_stays_within_the_rows(packed, known):
    # offsets outside of the rows, large and negative ones, as memory holds them that no plan has been written to
    n, cu = 300, [0, 100, 200, 300]
    leaves, g2 = tensors(n, 2, 2, 32, torch.float32), tensors(n, 2, 2, 32, torch.float32, seed=9)[:3]
    for wrong in ([2 ** 31 - 1, 7, -5], [-2 ** 31, -2 ** 31, 2 ** 31 - 1], [301, 5000, 2 ** 30], [0, 0, 0], [-1, -1, -1]):
        plan = packed.packed_plan(torch.tensor(cu, dtype=torch.int32, device="cuda"), n, max_seqlen=known)
        x = [t.detach().requires_grad_(True) for t in leaves]
        first = torch.autograd.grad(packed.packed_attention(*x[:3], plan), x[:3], x[3], create_graph=True)
        with torch.no_grad():
            plan.tensor.data[4] = wrong[0]
            plan.tensor.data[-6:-3] = torch.tensor(wrong, dtype=torch.int32)
        for t, like in zip(torch.autograd.grad(first, x, g2), x):
            assert t.shape == like.shape
        torch.cuda.synchronize()
