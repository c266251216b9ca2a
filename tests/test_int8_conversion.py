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
