"""Layer operators at the edges: results changed in place, exact zeros and projections beyond the range of f16 in gated blocks,
NaN in weights, second derivatives that are captured, of many tiles and of views, the benchmark's meta-step by relative size."""
import ctypes
import importlib
import math
import os
import sys

import pytest
import torch

from test_layers import (ACTIVATIONS, F32, HALF, PKG_DIR, SECOND, TYPES, capi, close, curve, curve_error, define_act, gated_inputs, inputs, layers, mm, near, norm_inputs,  # noqa: F401
                         passes, rounded, second)

CURVES = [a for a in ACTIVATIONS if a is not None]


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
