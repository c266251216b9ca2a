"""What the operators of kernels.int8_act refuse, on the host: the wrappers' checks on CPU tensors, which come before any
kernel, and the C entries' with addresses that nothing reads."""

from __future__ import annotations

import pytest
import torch

import kernels
from kernels import int8_act as a8

I8, BF, FP, F16 = torch.int8, torch.bfloat16, torch.float32, torch.float16
z = lambda *s, dt=FP: torch.zeros(*s, dtype=dt)


def _scaled(**over):
    a = {**dict(x=z(4, 32, dt=I8), sx=z(4), w=z(8, 32, dt=I8), sw=z(8), bias=None, dt=BF), **over}
    return a8.int8_scaled_matmul(a["x"], a["sx"], a["w"], a["sw"], a["bias"], out_dtype=a["dt"])


def _dynamic(**over):
    a = {**dict(x=z(4, 32), w=z(8, 32, dt=I8), sw=z(8), bias=None), **over}
    return a8.int8_dynamic_matmul(a["x"], a["w"], a["sw"], a["bias"])


SHARED = [(dict(w=z(8, 32)), TypeError), (dict(w=z(8, 33, dt=I8)), ValueError), (dict(w=z(32, dt=I8)), ValueError), (dict(sw=z(7)), ValueError),
          (dict(sw=z(8, dt=I8)), TypeError), (dict(sw=z(2, 2, 2)), ValueError), (dict(bias=z(7)), ValueError), (dict(bias=z(1, 8)), ValueError), (dict(bias=z(8, dt=I8)), TypeError),
          (dict(bias=z(8, dt=torch.float64)), TypeError), (dict(bias=z(8).requires_grad_()), ValueError), (dict(sw=z(8).requires_grad_()), ValueError),
          ({}, TypeError)]  # (the last: CPU tensors)


@pytest.mark.parametrize("over,error", SHARED + [
    (dict(x=z(4, 32)), TypeError), (dict(x=z(2, 2, 32, dt=I8)), ValueError), (dict(sx=z(3)), ValueError), (dict(sx=z(4, dt=I8)), TypeError),
    (dict(dt=torch.float64), TypeError), (dict(dt=torch.int32), TypeError), (dict(sx=z(4).requires_grad_()), ValueError),
    (dict(x=z(1, 131072, dt=I8), sx=z(1), w=z(8, 131072, dt=I8)), NotImplementedError)])
def test_scaled_matmul_refuses(over, error):
    with pytest.raises(error):
        _scaled(**over)


@pytest.mark.parametrize("over,error", SHARED + [(dict(x=z(4, 32, dt=I8)), TypeError), (dict(x=z(32)), ValueError), (dict(x=z(4, 32).requires_grad_()), ValueError),
                                                 (dict(x=z(4, 32, dt=torch.float64)), TypeError)])
def test_dynamic_matmul_refuses(over, error):
    with pytest.raises(error):
        _dynamic(**over)


@pytest.mark.parametrize("x,error", [(z(4, 32), TypeError), (z(4, 32, dt=I8), TypeError), (z(32), ValueError), (z(4, 32).requires_grad_(), ValueError)])
def test_quantize_rows_refuses(x, error):
    with pytest.raises(error):
        a8.quantize_rows(x)


@pytest.mark.parametrize("gate,up,error", [(z(4, 32), z(4, 33), ValueError), (z(4, 32), z(4, 32, dt=BF), ValueError), (z(4, 32, dt=I8), z(4, 32, dt=I8), TypeError),
                                           (z(32), z(32), ValueError), (z(4, 32), z(4, 32).requires_grad_(), ValueError), (z(4, 32), z(4, 32), TypeError)])
def test_silu_mul_quantize_refuses(gate, up, error):
    with pytest.raises(error):
        a8.silu_mul_quantize(gate, up)


@pytest.mark.parametrize("dh,q,s,error", [
    (z(4, 130), z(2, 4, 130, dt=I8), z(2, 4, 1), ValueError), (z(4, 130), z(2, 4, 129, dt=I8), z(2, 4, 2), ValueError),
    (z(4, 130), z(4, 2, 130, dt=I8), z(2, 4, 2), ValueError), (z(4, 130), z(2, 4, 130), z(2, 4, 2), TypeError), (z(4, 130), z(2, 4, 130, dt=I8), z(2, 4, 2, dt=F16), TypeError),
    (z(4, 130, dt=I8), z(2, 4, 130, dt=I8), z(2, 4, 2), TypeError), (z(130), z(2, 4, 130, dt=I8), z(2, 4, 2), ValueError),
    (z(4, 130).requires_grad_(), z(2, 4, 130, dt=I8), z(2, 4, 2), ValueError), (z(4, 130), z(2, 4, 130, dt=I8), z(2, 4, 2), TypeError)])
def test_silu_mul_backward_refuses(dh, q, s, error):
    with pytest.raises(error):
        a8.silu_mul_backward(dh, (q, s))


@pytest.mark.parametrize("dy,q,s,error", [
    (z(4, 8), z(4, 32), z(4), TypeError), (z(4, 8), z(5, 32, dt=I8), z(4), ValueError), (z(4, 8), z(4, 32, dt=I8), z(5), ValueError), (z(8), z(4, 32, dt=I8), z(4), ValueError),
    (z(4, 8), z(32, dt=I8), z(4), ValueError), (z(4, 8, dt=torch.float64), z(4, 32, dt=I8), z(4), TypeError), (z(4, 8).requires_grad_(), z(4, 32, dt=I8), z(4), ValueError),
    (z(4, 8), z(4, 32, dt=I8), z(4), TypeError)])
def test_weight_grad_refuses(dy, q, s, error):
    with pytest.raises(error):
        a8.int8_weight_grad(dy, q, s)


# ---------------------------------------------------------------- the C entries

GOOD = dict(x=1 << 20, sx=1 << 20, w=1 << 20, sw=1 << 20, bias=0, c=1 << 20, x_dt=-1, sw_dt=0, bias_dt=0, c_dt=2, ldx=64, ldw=64, ldc=32, M=4, N=32, K=64)


@pytest.mark.parametrize("over", [dict(M=-1), dict(N=-1), dict(K=0), dict(K=-4), dict(K=131072, ldx=131072, ldw=131072), dict(x=0), dict(w=0), dict(sw=0), dict(sx=0),
                                  dict(c=0), dict(x_dt=3), dict(sw_dt=2), dict(sw_dt=7), dict(c_dt=3), dict(bias=16, bias_dt=9), dict(ldx=63), dict(ldw=63), dict(ldc=31),
                                  dict(M=1 << 23), dict(N=1 << 23, ldc=1 << 23)])
def test_a8w8_entry_refuses(over):
    args = a8._ARGS.pack(*{**GOOD, **over}.values())
    assert kernels.lib().mlsx_a8w8(args, 1 << 20, 1 << 40, None) < 0


def test_a8w8_entry_refuses_workspaces():
    lib = kernels.lib()
    args = a8._ARGS.pack(*{**GOOD, "M": 200, "K": 60}.values())  # (rows that are no multiple of 16: copies)
    need = lib.mlsx_a8w8_ws(args)
    assert need > 0
    for at, n in ((0, need), (1 << 20, need - 1), ((1 << 20) + 8, need)):
        assert lib.mlsx_a8w8(args, at, n, None) == kernels.MLS_ERR_ARG
    assert lib.mlsx_a8w8(None, 0, 0, None) == kernels.MLS_ERR_ARG and lib.mlsx_a8w8_ws(None) == 0


def test_other_entries_refuse():
    lib, P = kernels.lib(), 1 << 20
    for a in ((P, 0, 8, -1, 8, P, 8, P, None), (P, 5, 8, 1, 8, P, 8, P, None), (0, 0, 8, 1, 8, P, 8, P, None), (P, 0, 7, 1, 8, P, 8, P, None), (P, 0, 8, 1, 8, P, 7, P, None),
              (P, 0, 8, 1, 8, P, 8, 0, None)):
        assert lib.mlsx_quantize_rows(*a) == kernels.MLS_ERR_ARG
    for a in ((P, 8, P, 8, 9, 1, 8, P, 8, P, 0, 0, None), (P, 7, P, 8, 0, 1, 8, P, 8, P, 0, 0, None), (P, 8, P, 8, 0, 1, 8, P, 8, P, P, 0, None),
              (P, 8, 0, 8, 0, 1, 8, P, 8, P, 0, 0, None), (P, 8, P, 8, 0, -1, 8, P, 8, P, 0, 0, None)):
        assert lib.mlsx_silu_mul_quantize(*a) == kernels.MLS_ERR_ARG
    for a in ((P, 8, 9, P, 8, 8, P, 1, 1, 1, 8, P, P, 8, None), (P, 7, 0, P, 8, 8, P, 1, 1, 1, 8, P, P, 8, None), (P, 8, 0, P, 8, 8, P, 0, 1, 1, 8, P, P, 8, None),
              (P, 8, 0, P, 8, 8, P, 1, 1, 1, 8, P, 0, 8, None)):
        assert lib.mlsx_silu_mul_backward(*a) == kernels.MLS_ERR_ARG
    need = lib.mlsx_dw_int8_workspace(2, 10, 8, 8)
    assert need > 0 and lib.mlsx_dw_int8_workspace(2, 0, 8, 8) == 0
    for a in ((P, 2, 8, P, 8, P, P, 8, 0, 8, 8, P, need, None), (P, 9, 8, P, 8, P, P, 8, 10, 8, 8, P, need, None), (P, 2, 7, P, 8, P, P, 8, 10, 8, 8, P, need, None),
              (P, 2, 8, P, 8, P, P, 8, 10, 8, 8, P, need - 1, None), (P, 2, 8, P, 8, P, P, 8, 10, 8, 8, P + 4, need, None), (0, 2, 8, P, 8, P, P, 8, 10, 8, 8, P, need, None)):
        assert lib.mlsx_dw_int8(*a) == kernels.MLS_ERR_ARG


def test_grids_past_32_bits_of_threads_are_refused():
    """Sizes whose operands no GPU here holds: an error of the entry's own before any launch."""
    lib, P = kernels.lib(), 1 << 20
    assert lib.mlsx_silu_mul_backward(P, 1 << 14, 0, P, 1 << 14, 1 << 38, P, 128, 1 << 31, 1 << 24, 1 << 14, P, P, 1 << 14, None) == kernels.MLS_ERR_UNSUPPORTED
    for K, ld in ((16, 16), (131071, 131071)):  # (tiles; rows to copy first)
        args = a8._ARGS.pack(P, P, P, P, 0, P, -1, 0, 0, 0, ld, ld, 1 << 22, 1 << 22, 1 << 22, K)
        assert lib.mlsx_a8w8(args, P, 1 << 60, None) == kernels.MLS_ERR_UNSUPPORTED
