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
