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
