"""More of what kernels.int8_act and the layers on it refuse and keep, on the host."""

from __future__ import annotations

import pytest
import torch

import kernels
from kernels import int8_act as a8


@pytest.mark.parametrize("dt", [torch.float64, torch.int8, torch.int32])
def test_weight_grad_refuses_other_output_types(dt):
    with pytest.raises(TypeError):
        a8.int8_weight_grad(torch.zeros(4, 8), torch.zeros(4, 32, dtype=torch.int8), torch.zeros(4), out_dtype=dt)


def test_weight_grad_entry_refuses_other_output_types():
    lib, P = kernels.lib(), 1 << 20
    need = lib.mlsx_dw_int8_workspace(2, 10, 8, 8)
    for dw_dt in (-1, 3, 7):
        assert lib.mlsx_dw_int8_to(P, 2, 8, P, 8, P, P, dw_dt, 8, 10, 8, 8, P, need, None) == kernels.MLS_ERR_ARG
    assert lib.mlsx_dw_int8_to(P, 2, 8, P, 8, P, P, 0, 7, 10, 8, 8, P, need, None) == kernels.MLS_ERR_ARG


@pytest.mark.parametrize("dy,kw,error", [(torch.zeros(4, 8), {}, TypeError), (torch.zeros(8), {}, ValueError), (torch.zeros(4, 8, dtype=torch.int8), {}, TypeError),
                                         (torch.zeros(4, 8), dict(out_dtype=torch.float64), TypeError), (torch.zeros(4, 8, requires_grad=True), {}, ValueError)])
def test_bias_grad_refuses(dy, kw, error):
    with pytest.raises(error):
        a8.bias_grad(dy, **kw)


def test_bias_grad_entry_refuses():
    lib, P = kernels.lib(), 1 << 20
    need = lib.mlsx_bias_grad_workspace(200, 30)
    assert need == 4 * 32 * 4 and lib.mlsx_bias_grad_workspace(64, 30) == 0 and lib.mlsx_bias_grad_workspace(0, 30) == 0
    for a in ((0, 0, 30, P, 0, 200, 30, P, need, None), (P, 5, 30, P, 0, 200, 30, P, need, None), (P, 0, 30, P, 5, 200, 30, P, need, None), (P, 0, 29, P, 0, 200, 30, P, need, None),
              (P, 0, 30, 0, 0, 200, 30, P, need, None), (P, 0, 30, P, 0, 0, 30, P, need, None), (P, 0, 30, P, 0, 200, -1, P, need, None), (P, 0, 30, P, 0, 200, 30, 0, 0, None),
              (P, 0, 30, P, 0, 200, 30, P, need - 1, None), (P, 0, 30, P, 0, 200, 30, P + 4, need, None)):
        assert lib.mlsx_bias_grad(*a) == kernels.MLS_ERR_ARG
    assert lib.mlsx_bias_grad(P, 0, 30, P, 0, 1 << 31, 30, P, 1 << 40, None) == kernels.MLS_ERR_UNSUPPORTED
