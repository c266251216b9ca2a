"""Input gradients of fp16 layers whose dy times the weights' scales lies below fp16's normal numbers, against 64 bits."""

from __future__ import annotations

import math

import pytest
import torch
import torch.nn as nn

from kernels.dequant_matmul import int8_dgrad
from train.int8 import Int8Linear, Int8SwiGLU

pytestmark = pytest.mark.gpu

F32, F16 = torch.float32, torch.float16
U = 2.0 ** -24


def cuda_gen(seed):
    return torch.Generator("cuda").manual_seed(seed)


def check_dx(dx, dy, q, s):
    """dy s is rounded to fp16 with the largest scale at [1/2, 1): off by half a step of 2^-10 relative, or half of 2^-24 of that unit. Then
    fp32 sums and one rounding to fp16. The weight-only product's kernels for few rows hold an INT8 weight as the fp16 1152 + q and take 1152 times the
    row's sum off again, so that their fp32 sums' roundings are of products by up to 1152 + |q|."""
    unit = 2.0 ** (math.floor(math.log2(float(s.float().max()))) + 1)
    p, w = dy.double().abs() * s.double(), q.double().abs()
    ref = (dy.double() * s.double()) @ q.double()
    tol = (p * 2.0 ** -11 + 2.0 ** -25 * unit) @ w + (2 * len(s) + 16) * U * (p @ (1152 + w)) + 2.0 ** -11 * ref.abs() + 2.0 ** -25
    off = (dx.double() - ref).abs()
    assert float(ref.abs().max()) < 65000
    assert bool((off <= tol).all()), float((off / tol).max())


# (rows: each of the weight-only product's routes)
@pytest.mark.parametrize("M", [1, 5, 16, 40, 256])
@pytest.mark.parametrize("N,K", [(64, 512), (65, 130), (256, 2048)])
@pytest.mark.parametrize("size", [1e-5, 1e-3, 1.0])
def test_dx_of_ordinary_weights(M, N, K, size):
    w = 0.02 * torch.randn(N, K, device="cuda", generator=cuda_gen(1))
    s = w.abs().amax(1) / 127
    q = torch.round(w / s[:, None]).to(torch.int8)
    dy = (size * torch.randn(M, N, device="cuda", generator=cuda_gen(2))).to(F16)
    check_dx(int8_dgrad(dy, q, s), dy, q, s)


@pytest.mark.parametrize("top", [1e-7, 1e-5, 1.0, 4000.0])
def test_dx_of_scales_of_every_size(top):
    """Scales up to `top` over 2^8, some rows of 1e-8; large ones whose products pass 65504 although dx does not."""
    q = torch.randint(-127, 128, (96, 200), device="cuda", dtype=torch.int8, generator=cuda_gen(1))
    s = top * torch.exp2(-8 * torch.rand(96, device="cuda", generator=cuda_gen(3)))
    s[5], s[::7] = top, 1e-8
    dy = torch.randn(30, 96, device="cuda", generator=cuda_gen(2)) * min(1e3, 1e-1 / top)
    if top == 4000.0:
        dy[:, 5] = 20.0
        q[5] = 0  # (8e4, which meets zeros)
    dy = dy.to(F16)
    check_dx(int8_dgrad(dy, q, s), dy, q, s)
    half = s.clamp(max=6e4).half()
    if bool((half > 0).all()):
        check_dx(int8_dgrad(dy, q, half), dy, q, half)


@pytest.mark.parametrize("size", [1e-5, 1e-3])
def test_fp16_linear_dx(size):
    torch.manual_seed(0)
    lin = nn.Linear(512, 256, bias=False)
    nn.init.normal_(lin.weight, std=0.02)
    layer = Int8Linear(lin.to("cuda", F16))
    x = torch.randn(100, 512, device="cuda").to(F16).requires_grad_()
    dy = (size * torch.randn(100, 256, device="cuda", generator=cuda_gen(2))).to(F16)
    dx, = torch.autograd.grad(layer(x), x, dy)
    from kernels.int8_act import quantize_rows
    check_dx(dx, dy, *quantize_rows(layer.weight.detach()))


def test_fp16_swiglu_gradients_are_their_torch_form():
    """dy of 1e-3 and weights of std 0.02. Each gradient passes at most four roundings to fp16 a side (a product's factor, dh, dgate or dup, the
    result) of 2^-11 relative to the norm at most, and dh, 3e-4, a grid of 2^-24: half of it, 2^-13 of dh. 12 * 2^-11 of the norm covers both sides."""
    D, H, M = 256, 512, 64
    torch.manual_seed(0)
    lins = [nn.Linear(D, H, bias=False), nn.Linear(D, H, bias=False), nn.Linear(H, D, bias=False)]
    for m in lins:
        nn.init.normal_(m.weight, std=0.02)
    x0 = 4 * torch.randn(M, D, generator=torch.Generator().manual_seed(1))
    dy = 1e-3 * torch.randn(M, D, generator=torch.Generator().manual_seed(2))
    out = []
    for k in (True, False):
        layer = Int8SwiGLU(*(m.to("cuda", F16) for m in lins), use_kernel=k)
        x = x0.to("cuda", F16).requires_grad_()
        out.append(torch.autograd.grad(layer(x), [x, *layer.parameters()], dy.to("cuda", F16)))
    for a, b in zip(*out):
        a, b = a.double(), b.double()
        assert float((a - b).norm()) <= 12 * 2.0 ** -11 * float(b.norm())


def test_replayed_over_scales_of_other_sizes():
    """The unit is found in the captured run: scales of other sizes, with eager calls and synchronizations between the replays."""
    q = torch.randint(-127, 128, (70, 130), device="cuda", dtype=torch.int8, generator=cuda_gen(1))
    dy, s = torch.zeros(33, 70, device="cuda", dtype=F16), torch.ones(70, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        int8_dgrad(dy, q, s)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = int8_dgrad(dy, q, s)
    for i, top in enumerate((1e-3, 5.0, 1e-8, 30.0)):
        d = (1e-2 * torch.randn(33, 70, device="cuda", generator=cuda_gen(i))).to(F16)
        t = top * (0.1 + torch.rand(70, device="cuda", generator=cuda_gen(9 + i)))
        dy.copy_(d)
        s.copy_(t)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, int8_dgrad(d, q, t))
        check_dx(out, d, q, t)
