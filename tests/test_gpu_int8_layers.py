"""train.int8 and QuantLinear(act_bits=8) on the kernels: they are what their operators give one after another, they agree with
their torch form, they train in a graph and serve."""

from __future__ import annotations

import pytest
import torch
import torch.nn as nn

from kernels import int8_act as a8
from kernels.dequant_matmul import int8_dgrad
from serve.quantize import Int8SwiGLU as ServeSwiGLU
from serve.quantize import QuantLinear, load_quantized, quantize_model, save_quantized
from train.int8 import Int8Linear, Int8SwiGLU, convert_linears_to_int8

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
U = 2.0 ** -24


def lins(dims, seed=0, bias=False, dtype=F32):
    torch.manual_seed(seed)
    return [nn.Linear(a, b, bias=bias).to("cuda", dtype) for a, b in dims]


@pytest.mark.parametrize("M,K,N", [(1, 64, 33), (40, 100, 130), (300, 512, 384)])
def test_linear_against_its_torch_form(M, K, N):
    """fp32: the same codes, so y is one sum's roundings off, and the gradients 2^-14 of the sum of their products' sizes
    (int8_dgrad takes dy as two bf16 parts, 2^-16; sums of up to 384 terms in fp32 on both sides, 2 * 384 * 2^-24)."""
    lin, = lins([(K, N)], bias=True)
    layers = [Int8Linear(lin, use_kernel=k) for k in (True, False)]
    xs = [torch.randn(M, K, device="cuda", generator=torch.Generator("cuda").manual_seed(1)).requires_grad_() for _ in layers]
    dy = torch.randn(M, N, device="cuda")
    ys = [l(x) for l, x in zip(layers, xs)]
    w, x = lin.weight.detach().abs(), xs[0].detach().abs()
    assert bool(((ys[0] - ys[1]).abs() <= 4 * U * (ys[1].abs() + x @ w.t())).all())
    a, b = (torch.autograd.grad(y, [x, l.weight, l.bias], dy) for y, x, l in zip(ys, xs, layers))
    # (an 8-bit value is at most 1 / 254 of its row's largest from the value itself: sizes by the largest)
    wide = lambda t: t + t.amax(1, keepdim=True) / 127
    for p, q, size in zip(a, b, (dy.abs() @ wide(w), dy.abs().t() @ wide(x), dy.abs().sum(0))):
        assert bool(((p - q).abs() <= 2.0 ** -14 * size).all())


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("M", [1, 16, 130])
def test_swiglu_is_its_operators_in_turn(M, dtype):
    D, H = 200, 520
    wg, wu, wd = lins([(D, H), (D, H), (H, D)], dtype=dtype)
    layer = Int8SwiGLU(wg, wu, wd)
    x = torch.randn(2, M, D, device="cuda").to(dtype).requires_grad_()
    y = layer(x)
    dy = torch.randn(2, M, D, device="cuda").to(dtype)
    got = torch.autograd.grad(y, [x, *layer.parameters()], dy)
    with torch.no_grad():
        ws = [a8.quantize_rows(m.weight) for m in (wg, wu, wd)]
        xq = a8.quantize_rows(x.reshape(-1, D))
        g, u = (a8.int8_scaled_matmul(*xq, *w, out_dtype=dtype) for w in ws[:2])
        hq, hs, kept = a8.silu_mul_quantize(g, u, checkpoint=True)
        assert torch.equal(y.reshape(-1, D), a8.int8_scaled_matmul(hq, hs, *ws[2], out_dtype=dtype))
        d = dy.reshape(-1, D)
        dg, du = a8.silu_mul_backward(int8_dgrad(d, *ws[2]), kept)
        dx = (int8_dgrad(dg, *ws[0]) + int8_dgrad(du, *ws[1])).reshape(x.shape)
        want = dx, a8.int8_weight_grad(dg, *xq), a8.int8_weight_grad(du, *xq), a8.int8_weight_grad(d, hq, hs)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_a_training_step_in_a_graph():
    """Forward, gradients and update captured once and replayed, against the same steps taken eagerly."""
    D, H, M = 128, 384, 64
    make = lambda: Int8SwiGLU(*lins([(D, H), (D, H), (H, D)], dtype=BF16))
    x, t = torch.randn(2, M, D, device="cuda", generator=torch.Generator("cuda").manual_seed(3)).to(BF16).unbind(0)

    def step(layer, x, t):
        ps = list(layer.parameters())
        gs = torch.autograd.grad((layer(x).float() - t.float()).square().mean(), ps)
        with torch.no_grad():
            for p, g in zip(ps, gs):
                p.sub_(g, alpha=0.5)

    eager, captured = make(), make()
    start = [p.detach().clone() for p in captured.parameters()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    sx, stt = x.clone(), t.clone()
    with torch.cuda.stream(side):
        step(captured, sx, stt)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(captured, sx, stt)
    with torch.no_grad():
        for p, s in zip(captured.parameters(), start):
            p.copy_(s)
    for i in range(4):
        xi, ti = torch.roll(x, i, 0), torch.roll(t, 2 * i, 0)
        sx.copy_(xi)
        stt.copy_(ti)
        graph.replay()
        torch.cuda.synchronize()
        step(eager, xi, ti)
        assert all(torch.equal(a, b) for a, b in zip(eager.parameters(), captured.parameters()))


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("M,N", [(1, 33), (300, 130), (5000, 257)])
def test_bias_gradient_eager_and_replayed(M, N, dtype):
    """Sums of M values that the matrix cores add in fp32, fp32's as three exact parts: 3 M roundings of the sum of sizes at most, then
    one to the type. A captured backward gives the same bits at each replay."""
    lin, = lins([(64, N)], bias=True, dtype=dtype)
    layer, x = Int8Linear(lin), torch.randn(M, 64, device="cuda").to(dtype)
    dys = [(torch.randn(M, N, device="cuda", generator=torch.Generator("cuda").manual_seed(i)) * 0.1).to(dtype) for i in range(4)]
    grads = lambda dy: torch.autograd.grad(layer(x), [layer.weight, layer.bias], dy)
    static = dys[0].clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        grads(static)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = grads(static)
    for dy in dys:
        static.copy_(dy)
        graph.replay()
        torch.cuda.synchronize()
        want = grads(dy)
        assert all(torch.equal(a, b) for a, b in zip(out, want))
        ref, size = dy.double().sum(0), dy.double().abs().sum(0)
        tol = 3 * M * U * size * (1 + torch.finfo(dtype).eps) + torch.finfo(dtype).eps / 2 * ref.abs() + 2.0 ** -25
        assert want[1].shape == (N,) and bool(((want[1].double() - ref).abs() <= tol).all())


def test_bias_gradient_of_no_tokens():
    layer = Int8Linear(lins([(64, 33)], bias=True)[0])
    layer(torch.zeros(0, 64, device="cuda")).sum().backward()
    assert layer.bias.grad.shape == (33,) and not bool(layer.bias.grad.any())


def test_convert_and_train_a_model():
    from test_gpu_layers import _Net
    torch.manual_seed(0)
    net = convert_linears_to_int8(_Net().cuda())
    assert any(isinstance(m, Int8SwiGLU) for m in net.modules()) and any(isinstance(m, Int8Linear) for m in net.modules())
    net(torch.randn(7, 30, 64, device="cuda")).square().mean().backward()
    assert all(bool(torch.isfinite(p.grad).all()) and bool(p.grad.any()) for p in net.parameters())


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_batches_of_no_tokens_and_expanded_gradients(dtype):
    layer = Int8SwiGLU(*lins([(64, 96), (64, 96), (96, 64)], dtype=dtype))
    x = torch.zeros(2, 0, 64, dtype=dtype, device="cuda", requires_grad=True)
    layer(x).sum().backward()
    assert x.grad.shape == x.shape and all(not bool(p.grad.any()) for p in layer.parameters())
    x = torch.randn(2, 5, 64, device="cuda").to(dtype)
    got = torch.autograd.grad(layer(x).sum(), layer.parameters())  # (a gradient of stride 0)
    y = layer(x)
    assert all(torch.equal(a, b) for a, b in zip(got, torch.autograd.grad(y, layer.parameters(), torch.ones_like(y))))


# ---------------------------------------------------------------- serving

@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("M", [1, 5, 16, 17, 200])
@torch.no_grad()
def test_quantlinear_act8(M, dtype):
    lin, = lins([(512, 384)])
    k, p = (QuantLinear(lin, use_kernel=u, act_bits=8) for u in (True, False))
    x = torch.randn(2, M, 512, device="cuda").to(dtype)
    y, want = k(x), p(x)
    # exact sums: two scales' roundings and one to the output's type, on each side
    half = torch.finfo(dtype).eps / 2
    assert y.dtype == dtype and bool(((y.double() - want.double()).abs() <= (4 * U + 2 * half) * want.double().abs()).all())


@pytest.mark.parametrize("M", [1, 16, 17, 200])
@torch.no_grad()
def test_served_swiglu_is_its_operators_in_turn(M):
    D, H = 256, 640
    qs = [QuantLinear(m, act_bits=8) for m in lins([(D, H), (D, H), (H, D)])]
    x = torch.randn(M, D, device="cuda").to(BF16)
    g, u = qs[0](x), qs[1](x)
    want = qs[2].matmul_codes(*a8.silu_mul_quantize(g, u), BF16)
    assert torch.equal(ServeSwiGLU(*qs)(x), want)
    assert ServeSwiGLU(*qs)(x[:0]).shape == (0, D)


@torch.no_grad()
def test_quantized_model_serves_and_round_trips(tmp_path):
    from test_host import _Model
    q = quantize_model(_Model().cuda(), act_bits=8)
    mlp, wq = q.blocks[0].mlp, q.blocks[0].attn.wq
    assert isinstance(mlp, ServeSwiGLU) and wq.act_bits == 8
    save_quantized(q, tmp_path / "q.safetensors")
    back = load_quantized(_Model(), tmp_path / "q.safetensors", device="cuda")
    x = torch.randn(3, mlp.w_gate.in_features, device="cuda")
    assert torch.equal(back.blocks[0].mlp(x), mlp(x)) and torch.equal(back.blocks[0].attn.wq(x), wq(x))


def test_serving_layers_refuse_gradients():
    lin, = lins([(64, 32)])
    with pytest.raises(ValueError):
        QuantLinear(lin, act_bits=8)(torch.randn(3, 64, device="cuda", requires_grad=True))
