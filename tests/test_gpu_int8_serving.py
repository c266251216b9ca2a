"""QuantLinear(act_bits=8) and Int8SwiGLU on the kernels: hooks, and forms that models meet."""

from __future__ import annotations

import pytest
import torch
import torch.nn as nn

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
