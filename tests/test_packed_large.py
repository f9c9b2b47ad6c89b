"""The packed operators on tensors of more than 2^31 elements: the last rows give what they give in a small call (GPU)."""
import importlib
import os
import sys

import pytest
import torch

PKG_DIR = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "610sample_b200")


@pytest.fixture(scope="module")
def modules():
    if PKG_DIR not in sys.path:
        sys.path.insert(0, PKG_DIR)
    return {n: importlib.import_module(n) for n in ("packed", "loss", "qk_prep")}


def filled(*shape, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(*shape, generator=g, device="cuda", dtype=torch.bfloat16)


@pytest.mark.gpu
def test_attention_rows_behind_2_to_the_31_elements(modules):
    packed = modules["packed"]
    H, D, n, last = 256, 128, 66000, 130
    cu = torch.cat([torch.arange(0, n - last, 659, device="cuda"), torch.tensor([n - last, n], device="cuda")]).to(torch.int32)
    q, do, k, v = filled(n, H, D), filled(n, H, D, seed=1), filled(n, 2, D, seed=2), filled(n, 2, D, seed=3)
    assert q.numel() > 2 ** 31
    plan = packed.packed_plan(cu, n)

    def passes(q, k, v, do, plan):
        q, k, v = (t.detach().requires_grad_(True) for t in (q, k, v))
        o = packed.packed_attention(q, k, v, plan)
        return [o.detach(), *torch.autograd.grad(o, (q, k, v), do)]
    got = [t[n - last:].clone() for t in passes(q, k, v, do, plan)]
    alone = packed.packed_plan(torch.tensor([0, last], dtype=torch.int32, device="cuda"), last)
    want = passes(*(t[n - last:].clone() for t in (q, k, v, do)), alone)
    for a, b in zip(got, want):      # the order of the sums may differ by the form of the kernel
        assert bool(((a - b).abs().float() <= 2 ** -7 * b.abs().float() + 1e-5 * float(b.abs().max())).all())


@pytest.mark.gpu
def test_norm_and_rotation_of_rows_behind_2_to_the_31_elements(modules):
    packed = modules["packed"]
    n, H, D, last = 132000, 128, 128, 50
    x = filled(n, H + 1, D)
    assert x.numel() > 2 ** 31
    w = filled(D, seed=1)
    pos = torch.arange(n, device="cuda", dtype=torch.int32) % 1000
    table = modules["qk_prep"].rope_table(D, 1000, device="cuda")

    def passes(x, pos):
        q, k = x[:, :H].detach().requires_grad_(True), x[:, H:].detach().requires_grad_(True)
        a, b = packed.packed_qk_norm_rope(q, k, w, w, table, pos)
        return [a.detach(), b.detach(), *torch.autograd.grad((a, b), (q, k), (x[:, :H], x[:, H:]))]
    got = [t[n - last:].clone() for t in passes(x, pos)]
    for a, b in zip(got, passes(x[n - last:].clone(), pos[n - last:].clone())):
        assert torch.equal(a, b)


@pytest.mark.gpu
def test_classes_behind_2_to_the_31_elements(modules):
    V, d, n = 1100000, 2000, 40
    w = filled(V, d)
    w *= 0.02
    assert w.numel() > 2 ** 31
    x = filled(n, d, seed=1)
    y = torch.arange(V - n, V, device="cuda")
    xl, wl = x.detach().requires_grad_(True), w.detach().requires_grad_(True)
    out = modules["loss"].linear_cross_entropy(xl, wl, y, reduction="sum")
    dx, dw = torch.autograd.grad(out, (xl, wl))
    lse = torch.full((n,), -float("inf"), device="cuda", dtype=torch.float64)
    want_dx = torch.zeros(n, d, device="cuda", dtype=torch.float64)
    for i in range(0, V, 100000):
        lse = torch.logaddexp(lse, torch.logsumexp(x.double() @ w[i:i + 100000].double().T, 1))
    for i in range(0, V, 100000):
        part = w[i:i + 100000].double()
        want_dx += torch.exp(x.double() @ part.T - lse[:, None]) @ part
    want_dx -= w[V - n:].double()
    tail = w[V - n:].double()
    G = torch.exp(x.double() @ tail.T - lse[:, None]) - torch.eye(n, device="cuda", dtype=torch.float64)
    assert abs(float(out.detach()) - float((lse - (x.double() * tail).sum(1)).sum())) <= 1e-4 * abs(float(out.detach()))
    # two roundings of 2^-8, of G and of the result, against the norm
    assert float((dx.double() - want_dx).norm() / want_dx.norm()) <= 2 ** -7
    want_dw = G.T @ x.double()
    assert float((dw[V - n:].double() - want_dw).norm() / want_dw.norm()) <= 2 ** -7
