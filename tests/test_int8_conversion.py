"""From trained INT8 models to served ones, and what conversion may change, on the host."""

from __future__ import annotations

import pytest
import torch
import torch.nn as nn
import torch.nn.functional as F

from serve.quantize import QuantLinear, load_quantized, quantize_model, save_quantized
from test_host import _Model  # toy model with the reference's slot names
from train.int8 import convert_linears_to_int8


def mlps(model):
    return [e for b in model.blocks for e in (b.mlp.experts if getattr(b, "is_moe", False) else [b.mlp])]


@pytest.mark.parametrize("kw", [dict(bits=8), dict(bits=4), dict(bits=8, act_bits=8)])
def test_a_trained_model_is_quantized_like_the_plain_one(kw, tmp_path):
    """Every MLP and projection runs, with the buffers that the unconverted model gives, and a checkpoint loads onto the converted model."""
    torch.manual_seed(0)
    m = _Model()
    c = convert_linears_to_int8(m, use_kernel=False)
    q, plain = quantize_model(c, use_kernel=False, **kw), quantize_model(m, use_kernel=False, **kw)
    assert list(q.state_dict()) == list(plain.state_dict())
    assert all(torch.equal(a, b) for a, b in zip(q.state_dict().values(), plain.state_dict().values()))
    save_quantized(q, tmp_path / "q.safetensors")
    back = load_quantized(convert_linears_to_int8(_Model(), use_kernel=False), tmp_path / "q.safetensors", use_kernel=False)
    x = torch.randn(5, m.blocks[0].mlp.w_gate.in_features)
    for a, b in zip(mlps(q), mlps(back)):
        assert all(isinstance(t, QuantLinear) for t in (a.w_gate, a.w_up, a.w_down))
        assert torch.equal(a(x), b(x))
        if "act_bits" not in kw:  # (which quantizes the product on its way)
            assert torch.equal(a(x), a.w_down(F.silu(a.w_gate(x)) * a.w_up(x)))
    for a, b in zip(q.blocks, back.blocks):
        assert torch.equal(a.attn.wq(x), b.attn.wq(x))


def test_other_modules_in_a_listed_place_are_refused(tmp_path):
    save_quantized(quantize_model(_Model(), use_kernel=False), tmp_path / "q.safetensors")
    m = _Model()
    m.blocks[0].attn.wq = nn.Identity()
    with pytest.raises(ValueError, match="not a linear layer"):
        load_quantized(m, tmp_path / "q.safetensors", use_kernel=False)
    c = convert_linears_to_int8(_Model(d=32), use_kernel=False)
    with pytest.raises(ValueError, match="stores"):
        load_quantized(c, tmp_path / "q.safetensors", use_kernel=False)


# ---------------------------------------------------------------- hooks

def hook_all(mlp, calls):
    def hook(name):
        return lambda m, args, out: calls.append((name, args[0].shape[0], out.shape[-1]))
    return [getattr(mlp, n).register_forward_hook(hook(n)) for n in ("w_gate", "w_up", "w_down")]


@pytest.mark.parametrize("rows", [1, 16, 17])
def test_hooks_on_projections_fire(rows):
    torch.manual_seed(0)
    m = _Model()
    mlp = m.blocks[0].mlp
    D, H = mlp.w_gate.in_features, mlp.w_gate.out_features
    x = torch.randn(rows, D)
    for e in (quantize_model(m, use_kernel=False, act_bits=8).blocks[0].mlp, convert_linears_to_int8(m, use_kernel=False).blocks[0].mlp):
        fused, calls = e(x), []
        handles = hook_all(e, calls)
        y = e(x)
        assert calls == [("w_gate", rows, H), ("w_up", rows, H), ("w_down", rows, D)]
        # (a code may be another where the product is rounded in between: 1 / 127 of the largest, once a weight's size)
        assert float((y - fused).detach().abs().max()) <= 0.02 * float(fused.detach().abs().max())
        for h in handles:
            h.remove()
        assert torch.equal(e(x), fused) and len(calls) == 3


def test_gradients_pass_hooked_projections():
    torch.manual_seed(0)
    e = convert_linears_to_int8(_Model(), use_kernel=False).blocks[0].mlp
    x, seen = torch.randn(9, e.w_gate.in_features, requires_grad=True), []
    want = torch.autograd.grad(e(x).sum(), [x, *e.parameters()])
    e.w_up.register_full_backward_hook(lambda m, gi, go: seen.append(go[0].shape))
    got = torch.autograd.grad(e(x).sum(), [x, *e.parameters()])
    assert seen == [(9, e.w_up.out_features)]
    # (here silu's own derivative meets gate and up in full width, there 8 bits of each group of 128)
    assert all(float((a - b).norm()) <= 0.05 * float(b.norm()) for a, b in zip(got, want))


# ---------------------------------------------------------------- modules with a SwiGLU's names that compute something else

class _Gated(nn.Module):
    def __init__(self, d=24, h=40, act=F.silu, drop=0.0):
        super().__init__()
        self.w_gate, self.w_up, self.w_down = nn.Linear(d, h, bias=False), nn.Linear(d, h, bias=False), nn.Linear(h, d, bias=False)
        self.act, self.drop = act, drop

    def forward(self, x):
        return self.w_down(F.dropout(self.act(self.w_gate(x)) * self.w_up(x), self.drop, self.training))


class _Swapped(_Gated):
    def forward(self, x):
        return self.w_down(F.silu(self.w_up(x)) * self.w_gate(x))


class _Scaled(_Gated):
    def __init__(self):
        super().__init__()
        self.scale = nn.Parameter(torch.full((), 2.0))

    def forward(self, x):
        return super().forward(x) * self.scale


class _Clipped(_Gated):
    def forward(self, x):
        return super().forward(x.clamp(-1, 1))


class _Rows(_Gated):
    """Its own way of writing it, with a module for the activation and rows flattened."""

    def __init__(self):
        super().__init__()
        self.fn = nn.SiLU()

    def forward(self, x):
        f = x.reshape(-1, x.shape[-1])
        up = self.w_up(f)
        return self.w_down(up * self.fn(self.w_gate(f))).reshape(x.shape)


class _Fp32Inside(_Gated):
    def forward(self, x):
        return self.w_down((F.silu(self.w_gate(x).float()) * self.w_up(x).float()).to(x.dtype))


class _Hook(_Gated):
    def __init__(self):
        super().__init__()
        self.register_forward_hook(lambda m, a, out: 3 * out)


class _Shell(nn.Module):
    def __init__(self, mlp):
        super().__init__()
        self.mlp = mlp

    def forward(self, x):
        return self.mlp(x)


class _Attn(nn.Module):
    def __init__(self, d):
        super().__init__()
        self.wq, self.wk, self.wv, self.wo = (nn.Linear(d, d, bias=False) for _ in range(4))


class _Blocks(nn.Module):
    def __init__(self, mlp):
        super().__init__()
        self.blocks = nn.ModuleList([_Shell(mlp)])
        self.blocks[0].attn = _Attn(24)


OTHERS = [lambda: _Gated(act=F.gelu), lambda: _Gated(act=torch.sigmoid), lambda: _Gated(drop=0.1), _Swapped, _Scaled, _Clipped, _Hook]


@pytest.mark.parametrize("make", OTHERS)
def test_conversion_keeps_what_other_mlps_compute(make):
    """Their linears are swapped, their forward is their own: the 8-bit operands are all that differs (a SwiGLU in their place is off by
    a tenth of the outputs and more)."""
    torch.manual_seed(0)
    m = _Blocks(make())
    x = 3 * torch.randn(50, 24)
    for c in (convert_linears_to_int8(m, use_kernel=False), quantize_model(m, use_kernel=False, act_bits=8)):
        mlp = c.blocks[0].mlp
        assert type(mlp) is type(m.blocks[0].mlp) and not isinstance(mlp.w_up, nn.Linear)
        torch.manual_seed(1)  # (dropout's)
        want = m.train().blocks[0](x)
        torch.manual_seed(1)
        got = c.train().blocks[0](x)
        assert float((got - want).detach().norm()) <= 0.03 * float(want.detach().norm())
    assert type(convert_linears_to_int8(make(), use_kernel=False)) is type(make())


def test_a_swiglu_by_another_name_is_fused(tmp_path):
    torch.manual_seed(0)
    state = torch.get_rng_state()
    for make in (_Rows, _Gated, _Fp32Inside):
        m = _Blocks(make()).eval()
        state = torch.get_rng_state()
        c, q = convert_linears_to_int8(m, use_kernel=False), quantize_model(m, use_kernel=False, act_bits=8)
        assert torch.equal(torch.get_rng_state(), state)  # (nothing drawn from the program's own generator)
        assert type(c.blocks[0].mlp).__name__ == type(q.blocks[0].mlp).__name__ == "Int8SwiGLU"
        assert not m.blocks[0].mlp.training and not c.blocks[0].mlp.training


def test_a_checkpoint_of_another_mlp_loads_as_it_was(tmp_path):
    torch.manual_seed(0)
    m = _Blocks(_Gated(act=F.gelu))
    q = quantize_model(m, use_kernel=False, act_bits=8)
    save_quantized(q, tmp_path / "q.safetensors")
    back = load_quantized(_Blocks(_Gated(act=F.gelu)), tmp_path / "q.safetensors", use_kernel=False)
    x = torch.randn(7, 24)
    assert type(back.blocks[0].mlp) is _Gated and torch.equal(back.blocks[0](x), q.blocks[0](x))


# ---------------------------------------------------------------- biases and ties

class _Biased(_Gated):
    def __init__(self):
        super().__init__()
        self.w_gate, self.w_up, self.w_down = nn.Linear(24, 40), nn.Linear(24, 40, bias=False), nn.Linear(40, 24)


def test_an_mlp_with_biases_becomes_three_linears():
    torch.manual_seed(0)
    m = _Blocks(_Biased())
    c = convert_linears_to_int8(m, use_kernel=False)
    mlp = c.blocks[0].mlp
    assert type(mlp) is _Biased and all(type(t).__name__ == "Int8Linear" for t in (mlp.w_gate, mlp.w_up, mlp.w_down))
    assert list(c.state_dict()) == list(m.state_dict()) and type(c.blocks[0].attn.wq).__name__ == "Int8Linear"
    x = torch.randn(50, 24)
    assert float((mlp(x) - m.blocks[0].mlp(x)).detach().norm()) <= 0.03 * float(m.blocks[0].mlp(x).detach().norm())


def test_ties_stay():
    """One layer in two places, one parameter in two layers, one MLP in two blocks and under two names: as in the model, so that
    gradients of all uses meet and an update reaches all."""
    torch.manual_seed(0)
    m = nn.Module()
    mlp = _Gated()
    m.a, m.b = _Blocks(mlp), _Blocks(mlp)
    m.a.blocks[0].again = mlp
    attn = m.a.blocks[0].attn
    attn.wk = attn.wq
    attn.wo.weight = attn.wv.weight
    m.embed = nn.Embedding(24, 24)
    m.b.blocks[0].attn.wq.weight = m.embed.weight
    m.out = nn.Linear(24, 24, bias=False)
    m.out.weight = m.embed.weight
    other = _Gated(act=F.gelu)
    other.w_up = other.w_gate
    m.other = other
    c = convert_linears_to_int8(m, use_kernel=False)
    blk, far = c.a.blocks[0], c.b.blocks[0]
    assert type(blk.mlp).__name__ == "Int8SwiGLU" and blk.mlp is far.mlp and blk.mlp is blk.again
    assert type(blk.attn.wq).__name__ == "Int8Linear" and blk.attn.wk is blk.attn.wq and blk.attn.wo.weight is blk.attn.wv.weight
    assert far.attn.wq.weight is c.embed.weight and c.out.weight is c.embed.weight
    assert c.other.w_up is c.other.w_gate and type(c.other.w_up).__name__ == "Int8Linear"
    assert len(list(c.parameters())) == len(list(m.parameters())) and list(c.state_dict()) == list(m.state_dict())
    assert not {id(p) for p in c.parameters()} & {id(p) for p in m.parameters()}
    x = torch.randn(5, 24)
    (blk.mlp(x) + far.mlp(x)).sum().backward()
    got = c.a.blocks[0].mlp.w_up.weight.grad
    c.zero_grad()
    far.mlp(x).sum().backward()
    assert torch.allclose(got, 2 * blk.mlp.w_up.weight.grad)


# ---------------------------------------------------------------- layers that serve have no gradient

def test_serving_layers_refuse_gradients_on_the_host():
    """Their scales carry a gradient in torch ops, which is no gradient of the layer."""
    torch.manual_seed(0)
    lin = QuantLinear(nn.Linear(24, 40, bias=False), use_kernel=False, act_bits=8)
    mlp = quantize_model(_Blocks(_Gated()), use_kernel=False, act_bits=8).blocks[0].mlp
    x = torch.randn(3, 24)
    for layer in (lin, mlp):
        with pytest.raises(ValueError):
            layer(x.clone().requires_grad_())
        with pytest.raises(ValueError):
            layer((2 * x.clone().requires_grad_()).reshape(1, 3, 24))
        with pytest.raises(ValueError), torch.autograd.forward_ad.dual_level():
            layer(torch.autograd.forward_ad.make_dual(x, torch.ones_like(x)))
        y = layer(x)
        with torch.no_grad():
            assert torch.equal(layer(x.clone().requires_grad_()), y)
    with pytest.raises(ValueError):
        lin.matmul_codes(torch.zeros(3, 24, dtype=torch.int8), torch.ones(3, requires_grad=True), torch.float32)
