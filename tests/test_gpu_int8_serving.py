"""QuantLinear(act_bits=8) and Int8SwiGLU on the kernels: hooks, and forms that models meet."""

from __future__ import annotations

import pytest
import torch
import torch.nn as nn

from kernels.int8_act import int8_scaled_matmul
from serve.quantize import Int8SwiGLU, QuantLinear

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows", [1, 8, 16, 17, 40])
@torch.no_grad()
def test_hooks_fire_at_every_batch_size(rows):
    torch.manual_seed(0)
    D, H = 64, 160
    e = Int8SwiGLU(*(QuantLinear(nn.Linear(a, b, bias=False).cuda(), act_bits=8) for a, b in ((D, H), (D, H), (H, D))))
    x, calls = torch.randn(rows, D, device="cuda"), []
    fused = e(x)
    handles = [m.register_forward_hook(lambda m, a, out: calls.append(out.shape)) for m in (e.w_gate, e.w_up, e.w_down)]
    y = e(x)
    assert calls == [(rows, H), (rows, H), (rows, D)]
    # a code may be another where the product is rounded in between: 1 / 127 of the largest, once a weight's size
    assert float((y - fused).abs().max()) <= 0.02 * float(fused.abs().max())
    for h in handles:
        h.remove()
    assert torch.equal(e(x), fused) and len(calls) == 3


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_sums_of_no_products_meet_their_scales(dtype):
    """K = 0: zero times the scales, so NaN where one is no finite number, as for any other sum of zero."""
    sx = torch.tensor([1.0, float("nan"), 2.0, float("inf")], device="cuda")
    sw = torch.tensor([0.5, float("-inf"), 3.0], device="cuda")
    bias = torch.tensor([1.5, 2.0, -4.0], device="cuda").to(dtype)
    for K in (0, 16):
        q, w = torch.zeros(4, K, dtype=torch.int8, device="cuda"), torch.zeros(3, K, dtype=torch.int8, device="cuda")
        for b in (None, bias):
            y = int8_scaled_matmul(q, sx, w, sw, b, out_dtype=dtype)
            bad = ~torch.isfinite(sx)[:, None] | ~torch.isfinite(sw)
            want = torch.zeros(4, 3, device="cuda") if b is None else b.float().expand(4, 3)
            assert y.dtype == dtype and torch.equal(torch.isnan(y), bad) and torch.equal(y[~bad].float(), want[~bad])


@pytest.mark.parametrize("kw", [dict(bits=8), dict(bits=4), dict(bits=8, act_bits=8)])
@torch.no_grad()
def test_a_trained_model_serves(kw, tmp_path):
    """Converted, quantized, stored and loaded on the device: the buffers and outputs of the model that was never converted."""
    from serve.quantize import load_quantized, quantize_model, save_quantized
    from test_host import _Model
    from train.int8 import convert_linears_to_int8
    torch.manual_seed(0)
    m = _Model().cuda()
    q, plain = quantize_model(convert_linears_to_int8(m), **kw), quantize_model(m, **kw)
    assert all(torch.equal(a, b) for a, b in zip(q.state_dict().values(), plain.state_dict().values()))
    save_quantized(q, tmp_path / "q.safetensors")
    back = load_quantized(convert_linears_to_int8(_Model()), tmp_path / "q.safetensors", device="cuda")
    x = torch.randn(5, m.blocks[0].mlp.w_gate.in_features, device="cuda")
    mlps = lambda n: [e for b in n.blocks for e in (b.mlp.experts if b.is_moe else [b.mlp])]
    for a, b, p in zip(mlps(q), mlps(back), mlps(plain)):
        want = p(x) if "act_bits" in kw else p.w_down(nn.functional.silu(p.w_gate(x)) * p.w_up(x))
        assert torch.equal(a(x), want) and torch.equal(b(x), want)
    for a, p in zip(q.blocks, plain.blocks):
        assert torch.equal(a.attn.wo(x), p.attn.wo(x))


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_layers_on_two_streams_at_once(dtype):
    """Two layers' forward and backward on streams of their own give what they give one after another."""
    from train.int8 import Int8Linear, Int8SwiGLU
    torch.manual_seed(0)
    lins = lambda *d: [nn.Linear(a, b, bias=False).to("cuda", dtype) for a, b in d]
    layers = [Int8SwiGLU(*lins((256, 640), (256, 640), (640, 256))), Int8Linear(nn.Linear(256, 384).to("cuda", dtype))]
    xs = [torch.randn(700, 256, device="cuda").to(dtype) for _ in layers]
    dys = [torch.randn(700, n, device="cuda").to(dtype) for n in (256, 384)]
    step = lambda l, x, dy: torch.autograd.grad(l(x), l.parameters(), dy)
    want = [step(*a) for a in zip(layers, xs, dys)]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in layers], [None, None]
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i] = step(layers[i], xs[i], dys[i])
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for g, w in zip(got, want) for a, b in zip(g, w))
