"""int8_weight_grad and the layers that use it where kept values leave 16-bit types' ranges, against 64 bits.

u = 2^-24 is half a step of fp32 relative to the value; eps / 2 half a step of a type."""

from __future__ import annotations

import math

import pytest
import torch
import torch.nn as nn

from kernels import int8_act as a8
from train.int8 import Int8Linear, Int8SwiGLU

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
U = 2.0 ** -24


def cuda_gen(seed):
    return torch.Generator("cuda").manual_seed(seed)


def some_codes(M, K, seed=0):
    return torch.randint(-127, 128, (M, K), device="cuda", dtype=torch.int8, generator=cuda_gen(seed))


def check_dw(dw, dy, q, s):
    """16-bit dy. A code times its scale's fraction is rounded to 11 bits: half a step of 2^-10 relative. dy with its scale's power of two is
    on a grid of 2^-24, at worst, where its column's largest has 2^14 by exponents, which products of fractions above 1/4 undercut by 4: half of it
    is 2^-37 of that largest. Then fp32 sums, and one rounding to the output's type."""
    d, v = dy.double().abs().t(), q.double().abs() * s.double()[:, None]
    ref = dy.double().t() @ (q.double() * s.double()[:, None])
    top = (d * s.double()).amax(1, keepdim=True)
    half, low = torch.finfo(dw.dtype).eps / 2, {F32: 2.0 ** -149, F16: 2.0 ** -25, BF16: 2.0 ** -133}[dw.dtype]
    err = 2.0 ** -11 * (d @ v) + 2.0 ** -37 * top * q.double().abs().sum(0) + (2 * len(dy) + 16) * U * (d @ v)
    off = (dw.double() - ref).abs()
    assert float(ref.abs().max()) < 65000  # (an fp16 result holds it)
    assert bool((off <= err * (1 + half) + half * ref.abs() + low).all()), float((off / (err + half * ref.abs() + low)).max())


@pytest.mark.parametrize("M,N,K", [(1, 3, 5), (60, 40, 33), (300, 128, 200)])
@pytest.mark.parametrize("top,size", [(1.2e5, 1e-3), (3e9, 1e-7), (6e4, 1e-3), (1.27e-6, 100.0), (3e-7, 1000.0), (6.0, 0.1)])
def test_fp16_weight_grad_of_scales_outside_its_range(M, N, K, top, size):
    """Kept values up to `top`: past 65504, and down to where fp16 has no bits left. Rows' scales spread over 2^6."""
    q = some_codes(M, K)
    s = top / 127 * torch.exp2(-6 * torch.rand(M, device="cuda", generator=cuda_gen(1)))
    s[M // 2] = top / 127
    dy = (size * torch.randn(M, N, device="cuda", generator=cuda_gen(2))).to(F16)
    check_dw(a8.int8_weight_grad(dy, q, s), dy, q, s)


def test_fp16_weight_grad_with_rows_of_zeros_and_one_far_above():
    """Scales of 1e-8 (rows of zeros) beside ordinary ones, and one row 2^17 above the others."""
    q, s = some_codes(100, 40), torch.full((100,), 0.05, device="cuda")
    q[::3], s[::3] = 0, 1e-8
    dy = (1e-2 * torch.randn(100, 30, device="cuda", generator=cuda_gen(2))).to(F16)
    check_dw(a8.int8_weight_grad(dy, q, s), dy, q, s)
    s[7] = 0.05 * 2 ** 17
    dy[7] *= 1e-2
    check_dw(a8.int8_weight_grad(dy, q, s), dy, q, s)
    q[:], s[:] = 0, 1e-8
    assert not bool(a8.int8_weight_grad(dy, q, s).any())


def test_fp16_swiglu_past_its_range_trains():
    """gate 400, up 300: the product is past 65504, the forward is finite, and so is every gradient, as in the torch form. The same codes on
    both sides (the values are exact), so the down projection's gradient differs by its roundings alone: 2^-11 of the sum of sizes and two
    to fp16."""
    D, H, M = 16, 64, 40
    torch.manual_seed(0)
    lins = [nn.Linear(D, H, bias=False), nn.Linear(D, H, bias=False), nn.Linear(H, D, bias=False)]
    with torch.no_grad():
        for lin, v in zip(lins, (4.0, 3.0)):
            lin.weight.zero_()
            lin.weight[:, 0] = v
            lin.weight[H // 2:, 0] = v / 64
        lins[2].weight.mul_(1e-2)
    x = torch.zeros(M, D)
    x[:, 0] = 100.0
    dy = 1e-3 * torch.randn(M, D, generator=torch.Generator().manual_seed(1))
    out = []
    for k in (True, False):
        layer = Int8SwiGLU(*(m.to("cuda", F16) for m in lins), use_kernel=k)
        xk = x.to("cuda", F16).requires_grad_()
        y = layer(xk)
        assert bool(torch.isfinite(y).all())
        out.append(torch.autograd.grad(y, [xk, *layer.parameters()], dy.to("cuda", F16)))
    assert all(bool(torch.isfinite(g).all()) for g in out[0])
    a, b = (o[3].double() for o in out)
    h = torch.full((M, H), 400.0 * 300.0, device="cuda", dtype=torch.float64)
    size = dy.cuda().double().abs().t() @ h
    assert float(b.abs().max()) > 100 and bool(((a - b).abs() <= 2.0 ** -10 * size + 2.0 ** -10 * b.abs()).all())


# ---------------------------------------------------------------- parameters of another type than the activations

@pytest.mark.parametrize("act,param", [(BF16, F32), (F16, F32), (F32, BF16), (F32, F16), (BF16, F16), (F16, BF16)])
@pytest.mark.parametrize("M,N,K", [(1, 33, 64), (300, 130, 65), (2000, 64, 48)])
def test_gradients_in_the_parameters_type(M, N, K, act, param):
    """fp32 sums rounded once, to the parameter's type; 16-bit dy meets the kept values rounded to 11 bits (half a step of 2^-10)."""
    torch.manual_seed(0)
    layer = Int8Linear(nn.Linear(K, N).to("cuda", param))
    x = torch.randn(M, K, device="cuda", generator=cuda_gen(1)).to(act)
    dy = (0.1 * torch.randn(M, N, device="cuda", generator=cuda_gen(2))).to(act)
    dw, db = torch.autograd.grad(layer(x), [layer.weight, layer.bias], dy)
    assert dw.dtype == db.dtype == param
    q, s = a8.quantize_rows(x)
    v = q.double() * s.double()[:, None]
    half, low = torch.finfo(param).eps / 2, {F32: 2.0 ** -149, F16: 2.0 ** -25, BF16: 2.0 ** -133}[param]
    for got, ref, size, factor in ((dw, dy.double().t() @ v, dy.double().abs().t() @ v.abs(), 0 if act == F32 else 2.0 ** -11),
                                   (db, dy.double().sum(0), dy.double().abs().sum(0), 0)):
        err = (factor + (3 * M + 16) * U) * size
        tol = err + half * (ref.abs() + err) + low
        off = (got.double() - ref).abs()
        assert bool((off <= tol).all()), float((off / tol).max())


def test_fp16_sums_past_its_range_reach_fp32_parameters():
    layer = Int8Linear(nn.Linear(16, 8).cuda())
    x, dy = torch.ones(2000, 16, device="cuda", dtype=F16), torch.full((2000, 8), 100.0, device="cuda", dtype=F16)
    dw, db = torch.autograd.grad(layer(x), [layer.weight, layer.bias], dy)
    assert torch.equal(db, torch.full_like(db, 2e5))
    # (one row's scale is 1 / 127 in fp32, its value 127 times that, rounded to fp16: within 2^-10 of 1)
    assert bool(((dw - 2e5).abs() <= 2e5 * 2.0 ** -10).all())


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("M,N,K", [(1, 3, 5), (300, 130, 65), (2100, 200, 333)])
def test_full_width_factors_on_request(M, N, K, dtype):
    """dy in fp32 with a 16-bit output: dy sx is rounded once, to fp32, and the result once."""
    q, s = some_codes(M, K), torch.rand(M, device="cuda", generator=cuda_gen(1)) + 0.1
    dy = (0.1 * torch.randn(M, N, device="cuda", generator=cuda_gen(2))).to(dtype)
    ref = dy.double().t() @ (q.double() * s.double()[:, None])
    size = dy.double().abs().t() @ (q.double().abs() * s.double()[:, None])
    tol = (3 * M + 16) * U * size * (1 + torch.finfo(dtype).eps) + torch.finfo(dtype).eps / 2 * ref.abs() + 2.0 ** -25
    dw = a8.int8_weight_grad(dy.float(), q, s, out_dtype=dtype)
    assert dw.dtype == dtype and bool(((dw.double() - ref).abs() <= tol).all())


def test_weight_grad_replayed_over_scales_of_other_sizes():
    q, s = some_codes(100, 40), torch.ones(100, device="cuda")
    dy = torch.zeros(100, 30, device="cuda", dtype=F16)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        a8.int8_weight_grad(dy, q, s)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = a8.int8_weight_grad(dy, q, s)
    for i, (top, size) in enumerate(((1e-3, 1.0), (900.0, 1e-3), (1e-8, 100.0), (5e6, 1e-6))):
        d = (size * torch.randn(100, 30, device="cuda", generator=cuda_gen(i))).to(F16)
        t = top * (0.1 + torch.rand(100, device="cuda", generator=cuda_gen(9 + i)))
        dy.copy_(d)
        s.copy_(t)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, a8.int8_weight_grad(d, q, t))
        check_dw(out, d, q, t)


@pytest.mark.parametrize("M,N,K", [(2100, 300, 200), (64, 2100, 130)])
@pytest.mark.parametrize("out", [F32, BF16])
def test_bf16_weight_grad_is_as_near_as_its_output(M, N, K, out):
    """Factors of 11 bits: their roundings, 2^-11 at most and 2^-12.8 in the mean square over a binade, fall at random, so that the sums are off by as
    much of the norm (1.4e-4; 3e-4 is the bound); bf16's own rounding of the result, 1.66e-3, grows by no more than a hundredth of itself."""
    q, _ = a8.quantize_rows(torch.randn(M, K, device="cuda", generator=cuda_gen(1)))
    s = 0.05 * torch.exp(0.5 * torch.randn(M, device="cuda", generator=cuda_gen(3)))
    dy = (1e-3 * torch.randn(M, N, device="cuda", generator=cuda_gen(2))).to(BF16)
    ref = dy.double().t() @ (q.double() * s.double()[:, None])
    off = lambda t: float((t.double() - ref).norm() / ref.norm())
    dw = a8.int8_weight_grad(dy, q, s, out_dtype=out)
    assert off(dw) <= (3e-4 if out == F32 else 1.02 * off(ref.to(BF16)))


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_gradients_of_every_size_in_a_column(dtype):
    """bf16 rows from 1e-30 to 1e30, fp16 from its smallest to its largest, masked tokens with scales far above the others, columns of zeros."""
    M, N, K = 200, 64, 48
    q, s = some_codes(M, K), torch.exp2(40 * torch.rand(M, device="cuda", generator=cuda_gen(1)) - 20)
    span = 90 if dtype == BF16 else 10
    dy = torch.randn(M, N, device="cuda", generator=cuda_gen(2)) * torch.exp2(span * (2 * torch.rand(1, N, device="cuda", generator=cuda_gen(3)) - 1))
    dy[::5] = 0
    s[::5] *= 2.0 ** 30
    dy[:, 7] = 0
    dy = dy.clamp(-6e4, 6e4).to(dtype) if dtype == F16 else dy.to(dtype)
    ref = dy.double().t() @ (q.double() * s.double()[:, None])
    d, v = dy.double().abs().t(), q.double().abs() * s.double()[:, None]
    err = (2.0 ** -11 + (2 * M + 16) * U) * (d @ v) + 2.0 ** -37 * (d * s.double()).amax(1, keepdim=True) * q.double().abs().sum(0)
    dw = a8.int8_weight_grad(dy, q, s, out_dtype=F32)
    assert not bool(dw[7].any()) and bool(((dw.double() - ref).abs() <= err + U * ref.abs() + 2.0 ** -149).all())
