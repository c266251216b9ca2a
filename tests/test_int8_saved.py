"""What train.int8's layers hold between forward and backward, by what gradients are asked for (on the host)."""

from __future__ import annotations

import itertools

import pytest
import torch
import torch.nn as nn

from train.int8 import Int8Linear, Int8SwiGLU

D, H, M = 40, 200, 16


def held(layer, x):
    kept = []
    with torch.autograd.graph.saved_tensors_hooks(lambda t: kept.append(t) or t, lambda t: t):
        y = layer(x)
    return y, kept


def codes(kept):
    return sorted(tuple(t.shape) for t in kept if t.dtype == torch.int8)


@pytest.mark.parametrize("x_needs,g,u,d", itertools.product((False, True), repeat=4))
def test_swiglu_holds_what_its_backward_reads(x_needs, g, u, d):
    """x's codes for gate and up, the product's for down, gate's and up's 8 bits and down's weight for what lies below them, gate's and up's weights
    for x: codes of every weight among them, 3 dim hidden bytes with all gradients."""
    torch.manual_seed(0)
    lins = [nn.Linear(D, H, bias=False), nn.Linear(D, H, bias=False), nn.Linear(H, D, bias=False)]
    layer = Int8SwiGLU(*lins, use_kernel=False)
    full = Int8SwiGLU(*lins, use_kernel=False)
    for m, need in zip((layer.w_gate, layer.w_up, layer.w_down), (g, u, d)):
        m.weight.requires_grad_(need)
    x = torch.randn(M, D)
    below = x_needs or g or u
    want = [(M, D)] * (g or u) + [(M, H)] * d + [(2, M, H), (D, H)] * below + [(H, D)] * 2 * x_needs
    y, kept = held(layer, x.clone().requires_grad_(x_needs))
    assert codes(kept) == sorted(want)
    # scales: fp32, one a row or group
    assert sum(t.numel() for t in kept if t.dtype != torch.int8) == M * (g or u) + M * d + (2 * M * 2 + D) * below + 2 * H * x_needs
    if not want:
        assert not y.requires_grad
        return
    xs = x.clone().requires_grad_()
    grads = torch.autograd.grad(full(xs).sum(), [xs, *full.parameters()])
    x2 = x.clone().requires_grad_(x_needs)
    layer(x2).sum().backward()
    got = [x2.grad, *(m.weight.grad for m in (layer.w_gate, layer.w_up, layer.w_down))]
    for a, b, need in zip(got, grads, (x_needs, g, u, d)):
        assert (a is not None) == need and (a is None or torch.equal(a, b))


@pytest.mark.parametrize("x_needs,w", itertools.product((False, True), repeat=2))
def test_linear_holds_what_its_backward_reads(x_needs, w):
    layer = Int8Linear(nn.Linear(D, H), use_kernel=False)
    layer.weight.requires_grad_(w)
    _, kept = held(layer, torch.randn(M, D, requires_grad=x_needs))
    assert codes(kept) == sorted([(H, D)] * x_needs + [(M, D)] * w)
