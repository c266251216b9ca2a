"""Activations in 8 bits (gfx950): the product of quantized activations and INT8 weights on the 8-bit matrix
cores, and the same codes as what a layer keeps for its backward pass.

The reference's INT8 path quantizes weights alone (kernels/dequant_matmul.py:17-25); nothing here has a
reference counterpart. Codes and scales are those of its weights, a row being a token:

    scale = max(max|row| / 127, 1e-8) in fp32, code = round-half-even(value / scale), int8

so kernels.int8_act.quantize_rows of a weight gives what serve.quantize.quantize_int8 gives. A row with an infinity or a NaN
has that as its scale and zeros as codes: its outputs are NaN, other rows are not touched.

    quantize_rows        x -> codes and scales
    int8_scaled_matmul   codes of x, INT8 weights -> y (sums are exact whole numbers)
    int8_dynamic_matmul  x, INT8 weights -> y: both of the above, for few rows in one launch
    silu_mul_quantize    gate, up -> codes of silu(gate) * up, and gate and up in 8 bits for the backward
    silu_mul_backward    gradients of gate and up from those
    int8_weight_grad     a weight's gradient from dy and the codes that its layer kept
    bias_grad            a bias's gradient

serve.quantize.QuantLinear(act_bits=8) serves with these, train.int8 trains with them. They have no
gradient of their own: inputs that ask for one are refused. The kernels are csrc/act8.hip, csrc/gemm_a8.hip and
csrc/gemm_dw8.hip.
"""

from __future__ import annotations

import struct

import torch
from torch.autograd import forward_ad

import kernels
from kernels._hip import _DT, dt_code
from kernels.paged_kv import _raw_stream, no_grad_of, one_device

_ARGS = struct.Struct("=6Q10q")  # mlsx_a8w8_args

GROUP = 128  # columns of gate and up that share a scale in a checkpoint
MAX_K = 131071  # the longest sum whose 32 bits hold products of -128 by -128


def _two(t: torch.Tensor, name: str, fn: str) -> torch.Tensor:
    """t with unit inner stride, its rows apart (copied where they are not)."""
    if t.dim() != 2:
        raise ValueError(f"{fn}: {name} must be 2-D, got shape {tuple(t.shape)}")
    if t.stride(1) != 1 or t.stride(0) < t.shape[1]:
        if t.shape[1] == 1 and t.stride(0) >= 1:
            return t.as_strided(t.shape, (t.stride(0), 1))
        t = t.contiguous()
    return t


def _codes(t: torch.Tensor, name: str, fn: str) -> torch.Tensor:
    if t.dtype != torch.int8:
        raise TypeError(f"{fn}: {name} must be int8, got {t.dtype}")
    return _two(t, name, fn)


def _scales(t: torch.Tensor, n: int, name: str, fn: str) -> torch.Tensor:
    """n scales as a dense vector: fp32 or fp16 as stored, other floats as fp32."""
    if t.numel() != n or t.dim() > 2:
        raise ValueError(f"{fn}: {name} has shape {tuple(t.shape)}, expected {n} scales")
    if t.dtype not in (torch.float32, torch.float16):
        if not t.dtype.is_floating_point:
            raise TypeError(f"{fn}: {name} must hold floats, got {t.dtype}")
        t = t.to(torch.float32)
    if t.dim() != 1:
        t = t.reshape(-1)
    return t if n <= 1 or t.stride(0) == 1 else t.contiguous()


def _on(dev: int, entry, *args) -> int:
    """entry(*args) with the tensors' device as the current one, whose kernels' limits the library sets."""
    if torch._C._cuda_getDevice() == dev:
        return entry(*args)
    with torch.cuda.device(dev):
        return entry(*args)


def _no_grad(fn: str, *tensors) -> None:
    if torch.is_grad_enabled() or forward_ad._current_level >= 0:
        no_grad_of(fn, *tensors)


def quantize_rows(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """x [M, K] (float32, float16, bfloat16) -> codes int8 [M, K], scales float32 [M]. The codes' rows
    are a multiple of 16 bytes apart."""
    fn = "quantize_rows"
    dt = dt_code(x.dtype, fn)
    x = _two(x, "x", fn)
    _no_grad(fn, x)
    dev = one_device(fn, x)
    M, K = x.shape
    q = torch.empty(M, -(-K // 16) * 16, dtype=torch.int8, device=x.device)
    s = torch.empty(M, dtype=torch.float32, device=x.device)
    kernels.check(_on(dev, kernels.lib().mlsx_quantize_rows, x.data_ptr(), dt, max(x.stride(0), K), M, K, q.data_ptr(), q.shape[1],
                      s.data_ptr(), _raw_stream(dev)), fn)
    return q[:, :K] if q.shape[1] != K else q, s


def _product(fn, x, sx, x_dt, w_q, sw, bias, out_dtype):
    """y [M, N] of codes (x_dt = -1, with scales sx) or values x."""
    M, K = x.shape
    w_q = _codes(w_q, "w_q", fn)
    N, Kw = w_q.shape
    if Kw != K:
        raise ValueError(f"{fn}: w_q {tuple(w_q.shape)} does not match K={K}")
    if K > MAX_K:
        raise NotImplementedError(f"{fn}: K={K}: sums of more than {MAX_K} products can pass 32 bits")
    sw = _scales(sw, N, "weight scales", fn)
    c_dt = dt_code(out_dtype, fn)
    b_at = b_dt = 0
    if bias is not None:
        if bias.dim() != 1 or bias.shape[0] != N:
            raise ValueError(f"{fn}: bias {tuple(bias.shape)}, expected ({N},)")
        b_dt = dt_code(bias.dtype, f"{fn} bias")
        if N > 1 and bias.stride(0) != 1:
            bias = bias.contiguous()
        b_at = bias.data_ptr()
    if torch.is_grad_enabled() or forward_ad._current_level >= 0:
        no_grad_of(fn, x, sx, sw, bias)
    dev = one_device(fn, x, w_q, sw, sx, bias)
    y = torch.empty(M, N, dtype=out_dtype, device=x.device)
    if M == 0 or N == 0:
        return y
    if K == 0:  # (no products: a sum of zero, times scales that may be no numbers)
        z = sw.float() * 0 if sx is None else sx[:, None] * 0 + sw.float() * 0
        return y.copy_((z if bias is None else z + bias.float()).expand(M, N))
    args = _ARGS.pack(x.data_ptr(), 0 if sx is None else sx.data_ptr(), w_q.data_ptr(), sw.data_ptr(), b_at, y.data_ptr(), x_dt,
                      _DT[sw.dtype], b_dt, c_dt, x.stride(0) if M > 1 else K, w_q.stride(0) if N > 1 else K, N, M, N, K)
    entry = kernels.lib().mlsx_a8w8
    rc = _on(dev, entry, args, 0, 0, _raw_stream(dev))
    if rc > 0:  # (the workspace that it needs)
        ws = torch.empty(rc, dtype=torch.uint8, device=x.device)
        rc = _on(dev, entry, args, ws.data_ptr(), rc, _raw_stream(dev))
    if rc:
        kernels.check(rc, fn)
    return y


def int8_scaled_matmul(x_q: torch.Tensor, sx: torch.Tensor, w_q: torch.Tensor, sw: torch.Tensor, bias: torch.Tensor | None = None,
                       *, out_dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """y[m, n] = (sum_k x_q[m, k] w_q[n, k]) sw[n] sx[m] + bias[n] in out_dtype.

    x_q int8 [M, K], sx [M]; w_q int8 [N, K], sw [N]; K up to MAX_K. The sum is exact; the scales, the bias and the
    rounding to out_dtype are applied to it in fp32. Any strides; K a multiple of 16 and rows 16-byte aligned
    save a copy of the operand."""
    fn = "int8_scaled_matmul"
    x_q = _codes(x_q, "x_q", fn)
    sx = _scales(sx, x_q.shape[0], "sx", fn)
    if sx.dtype != torch.float32:
        sx = sx.to(torch.float32)
    return _product(fn, x_q, sx, -1, w_q, sw, bias, out_dtype)


def int8_dynamic_matmul(x: torch.Tensor, w_q: torch.Tensor, sw: torch.Tensor, bias: torch.Tensor | None = None) -> torch.Tensor:
    """int8_scaled_matmul of quantize_rows(x), in x's dtype: a linear layer whose input is quantized per token as it comes."""
    fn = "int8_dynamic_matmul"
    dt = dt_code(x.dtype, fn)
    return _product(fn, _two(x, "x", fn), None, dt, w_q, sw, bias, x.dtype)


def silu_mul_quantize(gate: torch.Tensor, up: torch.Tensor, *, checkpoint: bool = False):
    """quantize_rows(silu(gate) * up), the product in fp32: (codes [M, H], scales [M]) for int8_scaled_matmul with a
    down projection. gate, up [M, H] of one dtype.

    checkpoint: also (codes int8 [2, M, H], scales float32 [2, M, ceil(H / GROUP)]) of gate and up, a
    scale for every GROUP columns, which silu_mul_backward reads. A NaN or infinity takes its group along."""
    fn = "silu_mul_quantize"
    if gate.shape != up.shape or gate.dtype != up.dtype:
        raise ValueError(f"{fn}: gate {tuple(gate.shape)} {gate.dtype} and up {tuple(up.shape)} {up.dtype} differ")
    dt = dt_code(gate.dtype, fn)
    gate, up = _two(gate, "gate", fn), _two(up, "up", fn)
    _no_grad(fn, gate, up)
    dev = one_device(fn, gate, up)
    M, H = gate.shape
    new = lambda *s, dtype: torch.empty(*s, dtype=dtype, device=gate.device)
    q = new(M, -(-H // 16) * 16, dtype=torch.int8)
    s = new(M, dtype=torch.float32)
    kept = (new(2, M, H, dtype=torch.int8), new(2, M, -(-H // GROUP), dtype=torch.float32)) if checkpoint else None
    kq, ks = (kept[0].data_ptr(), kept[1].data_ptr()) if checkpoint and H else (0, 0)
    kernels.check(_on(dev, kernels.lib().mlsx_silu_mul_quantize, gate.data_ptr(), max(gate.stride(0), H), up.data_ptr(),
                      max(up.stride(0), H), dt, M, H, q.data_ptr(), q.shape[1], s.data_ptr(), kq, ks, _raw_stream(dev)), fn)
    q = q[:, :H] if q.shape[1] != H else q
    return (q, s, kept) if checkpoint else (q, s)


def silu_mul_backward(dh: torch.Tensor, kept: tuple[torch.Tensor, torch.Tensor]) -> tuple[torch.Tensor, torch.Tensor]:
    """(dgate, dup) of h = silu(gate) * up in dh's dtype, from dh [M, H] and silu_mul_quantize's checkpoint:
    dup = dh g sig(g), dgate = dh u sig(g) (1 + g (1 - sig(g))), in fp32 from the 8-bit g and u."""
    fn = "silu_mul_backward"
    dt = dt_code(dh.dtype, fn)
    dh = _two(dh, "dh", fn)
    M, H = dh.shape
    q, s = kept
    G = -(-H // GROUP)
    if q.dtype != torch.int8 or s.dtype != torch.float32:
        raise TypeError(f"{fn}: a checkpoint holds int8 codes and float32 scales, got {q.dtype}, {s.dtype}")
    if q.shape != (2, M, H) or s.shape != (2, M, G):
        raise ValueError(f"{fn}: checkpoint {tuple(q.shape)}, {tuple(s.shape)}; expected {(2, M, H)}, {(2, M, G)} for dh {(M, H)}")
    q = q if q.stride(2) == 1 and q.stride(1) >= H else q.contiguous()
    s = s if s.stride(2) == 1 and s.stride(1) >= G else s.contiguous()
    _no_grad(fn, dh, s)
    dev = one_device(fn, dh, q, s)
    dgate, dup = (torch.empty(M, H, dtype=dh.dtype, device=dh.device) for _ in range(2))
    kernels.check(_on(dev, kernels.lib().mlsx_silu_mul_backward, dh.data_ptr(), max(dh.stride(0), H), dt, q.data_ptr(),
                      max(q.stride(1), H), q.stride(0), s.data_ptr(), max(s.stride(1), G), s.stride(0), M, H, dgate.data_ptr(),
                      dup.data_ptr(), H, _raw_stream(dev)), fn)
    return dgate, dup


def int8_weight_grad(dy: torch.Tensor, x_q: torch.Tensor, sx: torch.Tensor, *, out_dtype: torch.dtype | None = None) -> torch.Tensor:
    """dw [N, K] = dy [M, N]^T (x_q sx[:, None]) [M, K], fp32 sums rounded to out_dtype (None: dy's dtype): the gradient of a weight whose
    layer kept its input as quantize_rows' codes and scales. For 16-bit dy a kept value is rounded to 11 bits
    on the way to the matrix cores, and dy is not (but for numbers under 2^-32, fp16 2^-28, of its column's largest dy sx, which are on a grid of
    2^-39 of that); fp32 rounds dy * sx once, to fp32. Up to 2^20 tokens.

    int8_weight_grad(dy.float(), x_q, sx, out_dtype=dy.dtype) rounds the result alone to 16 bits, at three times the products."""
    fn = "int8_weight_grad"
    dt = dt_code(dy.dtype, fn)
    out_dtype = dy.dtype if out_dtype is None else out_dtype
    out_dt = dt_code(out_dtype, fn)
    dy, x_q = _two(dy, "dy", fn), _codes(x_q, "x_q", fn)
    (M, N), K = dy.shape, x_q.shape[1]
    if x_q.shape[0] != M:
        raise ValueError(f"{fn}: dy has {M} rows, x_q {x_q.shape[0]}")
    sx = _scales(sx, M, "sx", fn)
    if sx.dtype != torch.float32:
        sx = sx.to(torch.float32)
    _no_grad(fn, dy, sx)
    dev = one_device(fn, dy, x_q, sx)
    dw = torch.empty(N, K, dtype=out_dtype, device=dy.device)
    if M == 0:
        return dw.zero_()
    if N == 0 or K == 0:
        return dw
    lib = kernels.lib()
    need = lib.mlsx_dw_int8_workspace(dt, M, N, K)
    ws = torch.empty(need, dtype=torch.uint8, device=dy.device)
    kernels.check(_on(dev, lib.mlsx_dw_int8_to, dy.data_ptr(), dt, max(dy.stride(0), N), x_q.data_ptr(), max(x_q.stride(0), K),
                      sx.data_ptr(), dw.data_ptr(), out_dt, K, M, N, K, ws.data_ptr(), need, _raw_stream(dev)), fn)
    return dw


def bias_grad(dy: torch.Tensor, *, out_dtype: torch.dtype | None = None) -> torch.Tensor:
    """db [N] = dy [M, N] summed over its rows, fp32 sums rounded to out_dtype (None: dy's dtype), in an order that the sizes alone decide. torch's
    own sum over many rows clears memory with a memset, which a captured graph must not hold."""
    fn = "bias_grad"
    dt = dt_code(dy.dtype, fn)
    out_dtype = dy.dtype if out_dtype is None else out_dtype
    out_dt = dt_code(out_dtype, fn)
    dy = _two(dy, "dy", fn)
    _no_grad(fn, dy)
    dev = one_device(fn, dy)
    M, N = dy.shape
    db = torch.empty(N, dtype=out_dtype, device=dy.device)
    if M == 0:
        return db.zero_()
    lib = kernels.lib()
    need = lib.mlsx_bias_grad_workspace(M, N)
    ws = torch.empty(need, dtype=torch.uint8, device=dy.device)
    kernels.check(_on(dev, lib.mlsx_bias_grad, dy.data_ptr(), dt, max(dy.stride(0), N), db.data_ptr(), out_dt, M, N, ws.data_ptr(), need,
                      _raw_stream(dev)), fn)
    return db
