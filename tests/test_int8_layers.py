"""train.int8 and QuantLinear(act_bits=8) in torch ops on the host: what they compute, keep, convert, store and refuse."""

from __future__ import annotations

import pytest
import torch
import torch.nn as nn

from serve.quantize import Int8SwiGLU as ServeSwiGLU
from serve.quantize import QuantLinear, load_quantized, quantize_int8, quantize_model, save_quantized
from test_host import _Model  # toy model with the reference's slot names
from train.int8 import Int8Linear, Int8SwiGLU, convert_linears_to_int8

D, H = 40, 200
U = 2.0 ** -24


def values(t):
    """t as its 8-bit form gives it back, a scale a row, in 64 bits."""
    q, s = quantize_int8(t.detach())
    return q.double() * s.double()[:, None]


def kept(t):
    """t as a checkpoint gives it back, a scale for every 128 columns."""
    return torch.cat([values(p) for p in t.split(128, 1)], 1)


def mlp(seed=0):
    torch.manual_seed(seed)
    return [nn.Linear(D, H, bias=False), nn.Linear(D, H, bias=False), nn.Linear(H, D, bias=False)]


def test_linear_is_straight_through():
    torch.manual_seed(0)
    lin = nn.Linear(D, 24)
    layer = Int8Linear(lin, use_kernel=False)
    x = torch.randn(2, 7, D, requires_grad=True)
    y = layer(x)
    f = x.reshape(-1, D)
    want = values(f) @ values(lin.weight).t() + lin.bias.double()
    assert y.shape == (2, 7, 24) and torch.allclose(y.reshape(-1, 24).double(), want, rtol=U, atol=0)
    dy = torch.randn_like(y)
    dx, dw, db = torch.autograd.grad(y, [x, layer.weight, layer.bias], dy)
    d = dy.reshape(-1, 24).double()
    # fp32 sums of 24 and 14 products of factors that are rounded once: 32 u of the sum of their sizes
    close = lambda a, b, size: bool(((a.double() - b).abs() <= 32 * U * size).all())
    assert close(dx.reshape(-1, D), d @ values(lin.weight), d.abs() @ values(lin.weight).abs())
    assert close(dw, d.t() @ values(f), d.abs().t() @ values(f).abs())
    assert close(db, d.sum(0), d.abs().sum(0))


def test_swiglu_uses_what_it_kept():
    lins = mlp()
    layer = Int8SwiGLU(*lins, use_kernel=False)
    x = torch.randn(9, D, requires_grad=True)
    y = layer(x)
    g, u = (values(x) @ values(m.weight).t() for m in lins[:2])
    g, u = g.float(), u.float()
    h = values(g * torch.sigmoid(g) * u)
    wg, wu, wd = (values(m.weight) for m in lins)
    assert torch.allclose(y.double(), h @ wd.t(), rtol=1e-6, atol=1e-7)
    dy = torch.randn_like(y)
    got = torch.autograd.grad(y, [x, layer.w_gate.weight, layer.w_up.weight, layer.w_down.weight], dy)
    d = dy.double()
    gk, uk = kept(g).requires_grad_(), kept(u).requires_grad_()
    dg, du = torch.autograd.grad(gk * torch.sigmoid(gk) * uk, [gk, uk], d @ wd)
    for a, b in zip(got, (dg @ wg + du @ wu, dg.t() @ values(x), du.t() @ values(x), d.t() @ h)):
        # fp32 sums of up to 200 products against 64 bits: a few 2^-24 of the largest
        assert float((a.double() - b).abs().max()) <= 200 * U * float(b.abs().max())


def test_what_is_kept_is_8_bits():
    layer = Int8SwiGLU(*mlp(), use_kernel=False)
    x = torch.randn(16, D)
    held = []
    with torch.autograd.graph.saved_tensors_hooks(lambda t: held.append(t) or t, lambda t: t):
        layer(x)
    activations = [t for t in held if t.dtype == torch.int8 and t.shape[-1] in (D, H) and 16 in t.shape]
    assert sum(t.numel() for t in activations) == 16 * (D + 3 * H)
    assert all(t.dtype == torch.int8 or t.numel() <= 4 * max(D, H, 16) for t in held)


def test_gradients_that_nobody_asks_for_are_not_made():
    layer = Int8SwiGLU(*mlp(), use_kernel=False).requires_grad_(False)
    x = torch.randn(3, D, requires_grad=True)
    layer(x).sum().backward()
    assert x.grad is not None and layer.w_gate.weight.grad is None
    assert not layer(x.detach()).requires_grad
    lin = Int8Linear(nn.Linear(D, 8, bias=False), use_kernel=False)
    lin(x.detach()).sum().backward()
    assert lin.weight.grad is not None


def test_no_checkpoint_without_gradients(monkeypatch):
    import train.int8 as t8
    kept, made = [], t8._silu_mul
    monkeypatch.setattr(t8, "_silu_mul", lambda *a: kept.append(a[3]) or made(*a))
    layer, x = Int8SwiGLU(*mlp(), use_kernel=False), torch.randn(3, D)
    y = layer(x)
    with torch.no_grad():
        z = layer(x)
    with torch.inference_mode():
        layer(x)
    assert kept == [True, False, False] and torch.equal(y, z) and not z.requires_grad


def test_frozen_parameters_stay_frozen():
    lin = nn.Linear(D, 8)
    lin.weight.requires_grad_(False)
    layer = Int8Linear(lin, use_kernel=False)
    assert not layer.weight.requires_grad and layer.bias.requires_grad
    w = mlp()
    w[1].requires_grad_(False)
    swi = Int8SwiGLU(*w, use_kernel=False)
    assert [m.weight.requires_grad for m in (swi.w_gate, swi.w_up, swi.w_down)] == [True, False, True]
    swi(torch.randn(3, D)).sum().backward()
    assert swi.w_up.weight.grad is None and swi.w_gate.weight.grad is not None
    c = convert_linears_to_int8(_Model().requires_grad_(False), use_kernel=False)
    assert not any(p.requires_grad for p in c.parameters())


def test_second_derivatives_are_refused():
    layer = Int8Linear(nn.Linear(D, 8), use_kernel=False)
    x = torch.randn(3, D, requires_grad=True)
    g, = torch.autograd.grad(layer(x).square().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_dtypes_and_empty_batches(dtype):
    layer = Int8SwiGLU(*mlp(), use_kernel=False)  # (fp32 parameters)
    x = torch.randn(5, D).to(dtype).requires_grad_()
    y = layer(x)
    y.sum().backward()
    assert y.dtype == dtype and x.grad.dtype == dtype and layer.w_up.weight.grad.dtype == torch.float32
    with pytest.raises(ValueError):
        Int8SwiGLU(nn.Linear(D, H), *mlp()[1:])


def test_convert_keeps_names_and_weights():
    m = _Model()
    c = convert_linears_to_int8(m, use_kernel=False)
    assert list(c.state_dict()) == list(m.state_dict())
    assert all(torch.equal(a, b) for a, b in zip(c.state_dict().values(), m.state_dict().values()))
    blk = c.blocks[0]
    assert isinstance(blk.attn.wq, Int8Linear) and isinstance(blk.mlp, Int8SwiGLU)
    assert isinstance(m.blocks[0].attn.wq, nn.Linear)
    for b in c.blocks:
        if getattr(b, "is_moe", False):
            assert all(isinstance(e, Int8SwiGLU) for e in b.mlp.experts)


# ---------------------------------------------------------------- QuantLinear(act_bits=8)

def test_quantlinear_act8_host():
    torch.manual_seed(1)
    lin = nn.Linear(D, 24, bias=False)
    q = QuantLinear(lin, bits=8, use_kernel=False, act_bits=8)
    x = torch.randn(2, 3, D)
    y = q(x)
    assert torch.allclose(y.reshape(-1, 24).double(), values(x.reshape(-1, D)) @ values(lin.weight).t(), rtol=U, atol=0)
    assert torch.equal(QuantLinear.from_quantized(q.w_q, q.scale, 8, 32, D, False, act_bits=8)(x), y)
    assert QuantLinear(lin, use_kernel=False).act_bits is None


@pytest.mark.parametrize("kw", [dict(bits=4, act_bits=8), dict(bits=8, act_bits=4), dict(bits=8, act_bits=16)])
def test_act_bits_refuses(kw):
    with pytest.raises(ValueError):
        QuantLinear(nn.Linear(64, 64, bias=False), use_kernel=False, **kw)
    with pytest.raises(ValueError):
        quantize_model(_Model(), use_kernel=False, **kw)


def test_quantized_model_is_fused_and_round_trips(tmp_path):
    m = _Model()
    q = quantize_model(m, bits=8, use_kernel=False, act_bits=8)
    plain = quantize_model(m, bits=8, use_kernel=False)
    assert list(q.state_dict()) == list(plain.state_dict())
    mlps = [e for b in q.blocks for e in (b.mlp.experts if getattr(b, "is_moe", False) else [b.mlp])]
    assert all(isinstance(e, ServeSwiGLU) for e in mlps)
    assert not any(isinstance(x, ServeSwiGLU) for x in plain.modules())
    x = torch.randn(5, q.blocks[0].mlp.w_gate.in_features)
    e = q.blocks[0].mlp
    g, u = (values(x) @ (w.w_q.double() * w.scale.double()[:, None]).t() for w in (e.w_gate, e.w_up))
    g, u = g.float(), u.float()
    want = values(g * torch.sigmoid(g) * u) @ (e.w_down.w_q.double() * e.w_down.scale.double()[:, None]).t()
    assert torch.allclose(e(x).double(), want, rtol=1e-6, atol=1e-7)
    path = tmp_path / "q.safetensors"
    save_quantized(q, path)
    back = load_quantized(_Model(), path, use_kernel=False)
    assert isinstance(back.blocks[0].mlp, ServeSwiGLU) and back.blocks[0].attn.wq.act_bits == 8
    assert torch.equal(back.blocks[0].mlp(x), e(x))
    save_quantized(plain, path)
    assert load_quantized(_Model(), path, use_kernel=False).blocks[0].attn.wq.act_bits is None
    with pytest.raises(ValueError):
        save_quantized(q, path, {"a:x": "8"})
    with pytest.raises(ValueError):
        ServeSwiGLU(plain.blocks[0].mlp.w_gate, e.w_up, e.w_down)
