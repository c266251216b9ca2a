"""INT8 training layers whose activations live in 8 bits, on the gfx950 kernels (no reference counterpart; its
INT8 estimator, kernels/autograd_ops.py:95-134, quantizes the weight alone and keeps x in full width).

Forward: the weight (per output row) and the input (per token) are quantized, and their codes meet on the 8-bit
matrix cores. What a layer keeps for its backward is those codes: a quarter of fp32's bytes, half of 16-bit types'.
Backward, straight through both quantizers: dx = dy times the quantized weight, dw = dy^T times the kept codes,
each operand the one that the forward used, with fp32 sums; dw in the parameter's type. On the kernels one factor of a product is
rounded for the matrix cores: 16-bit dx to dy's type (dy times a weight's scale), 16-bit dw to 11 bits (a code times a token's), fp32 dx to two bf16
parts (2^-16).

Int8SwiGLU is a whole MLP, w_down(silu(w_gate(x)) * w_up(x)): the product goes to w_down as codes made in the
kernel that computes it, and gate and up are kept in 8 bits with a scale for every 128 columns. For a batch of M
tokens it keeps M (dim + 3 hidden) bytes and scales, where the plain layers keep M (dim + 3 hidden) values and silu's own; and until the
backward the weights' codes, 3 dim hidden bytes, where the plain layers have the parameters themselves. What no wanted gradient reads is not kept.

A backward takes up to 2^20 tokens at a time (int8_weight_grad).

In a captured graph take gradients with torch.autograd.grad, or capture before any eager backward of the same
parameters: torch's accumulation into .grad stays on the stream where a parameter was first used.

use_kernel=False computes the same in torch ops, on the host or a device, with those factors in fp32.
"""

from __future__ import annotations

import torch
import torch.nn as nn
from torch.autograd.function import once_differentiable

from serve.quantize import computes_swiglu, has_hooks, quantize_int8

_GROUP = 128
_ATTN, _MLP = ("wq", "wk", "wv", "wo"), ("w_gate", "w_up", "w_down")


def _rows(x, use_kernel):
    """Codes and scales of x's rows."""
    if use_kernel:
        from kernels.int8_act import quantize_rows
        return quantize_rows(x)
    return quantize_int8(x.float())


def _matmul(x_q, sx, w_q, sw, bias, dtype, use_kernel):
    if use_kernel:
        from kernels.int8_act import int8_scaled_matmul
        return int8_scaled_matmul(x_q, sx, w_q, sw, bias, out_dtype=dtype)
    y = (x_q.double() @ w_q.double().t()) * sw.double() * sx.double()[:, None]
    return (y if bias is None else y + bias.double()).to(dtype)


def _input_grad(dy, w_q, sw, use_kernel):
    if use_kernel:
        from kernels.dequant_matmul import int8_dgrad
        return int8_dgrad(dy, w_q, sw)
    return (dy.float() @ (w_q.float() * sw.float()[:, None])).to(dy.dtype)


def _weight_grad(dy, x_q, sx, use_kernel, dtype):
    if use_kernel:
        from kernels.int8_act import int8_weight_grad
        return int8_weight_grad(dy, x_q, sx, out_dtype=dtype)
    return (dy.float().t() @ (x_q.float() * sx[:, None])).to(dtype)


def _bias_grad(dy, use_kernel, dtype):
    if use_kernel:
        from kernels.int8_act import bias_grad
        return bias_grad(dy, out_dtype=dtype)
    return dy.sum(0, dtype=torch.float32).to(dtype)


def _silu_mul(g, u, use_kernel, keep):
    """Codes and scales of silu(g) * u, and gate and up in 8 bits where they are kept."""
    if use_kernel:
        from kernels.int8_act import silu_mul_quantize
        return silu_mul_quantize(g, u, checkpoint=True) if keep else (*silu_mul_quantize(g, u), None)
    M, H = g.shape
    g, u = g.float(), u.float()
    kept = None
    if keep:
        pad = nn.functional.pad(torch.stack([g, u]), (0, -H % _GROUP))
        q, s = quantize_int8(pad.reshape(-1, _GROUP))
        kept = q.reshape(2, M, -1)[..., :H], s.reshape(2, M, -1)
    return *quantize_int8(g * torch.sigmoid(g) * u), kept


def _silu_mul_grad(dh, kept, use_kernel):
    if use_kernel:
        from kernels.int8_act import silu_mul_backward
        return silu_mul_backward(dh, kept)
    q, s = kept
    g, u = q.float() * s.repeat_interleave(_GROUP, 2)[..., :q.shape[2]]
    d, sig = dh.float(), torch.sigmoid(g)
    return (d * u * sig * (1 + g * (1 - sig))).to(dh.dtype), (d * g * sig).to(dh.dtype)


class _Int8LinearFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w, bias, use_kernel):
        w_q, sw = _rows(w, use_kernel)
        x_q, sx = _rows(x, use_kernel)
        ctx.use_kernel, ctx.dtypes = use_kernel, (w.dtype, None if bias is None else bias.dtype)
        need_x, need_w = ctx.needs_input_grad[:2]
        ctx.save_for_backward(*((w_q, sw) if need_x else (None, None)), *((x_q, sx) if need_w else (None, None)))
        return _matmul(x_q, sx, w_q, sw, bias, x.dtype, use_kernel)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        w_q, sw, x_q, sx = ctx.saved_tensors
        need_x, need_w, need_b = ctx.needs_input_grad[:3]
        wt, bt = ctx.dtypes
        dx = _input_grad(dy, w_q, sw, ctx.use_kernel) if need_x else None
        dw = _weight_grad(dy, x_q, sx, ctx.use_kernel, wt) if need_w else None
        return dx, dw, _bias_grad(dy, ctx.use_kernel, bt) if need_b else None, None


class _Int8SwiGLUFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w_gate, w_up, w_down, use_kernel, grad):
        # (grad: the caller's grad mode; needs_input_grad does not know of it)
        need_x, need_g, need_u, need_d = (grad and n for n in ctx.needs_input_grad[:4])
        below = need_x or need_g or need_u  # a gradient that comes through down's
        weights = [_rows(w, use_kernel) for w in (w_gate, w_up, w_down)]
        x_q, sx = _rows(x, use_kernel)
        g, u = (_matmul(x_q, sx, *w, None, x.dtype, use_kernel) for w in weights[:2])
        h_q, sh, kept = _silu_mul(g, u, use_kernel, below)
        ctx.use_kernel, ctx.dtypes = use_kernel, (w_gate.dtype, w_up.dtype, w_down.dtype)
        none = None, None
        ctx.save_for_backward(*((x_q, sx) if need_g or need_u else none), *((h_q, sh) if need_d else none), *(kept if below else none),
                              *(weights[0] + weights[1] if need_x else none + none), *(weights[2] if below else none))
        return _matmul(h_q, sh, *weights[2], None, x.dtype, use_kernel)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x_q, sx, h_q, sh, kq, ks, gq, gs, uq, us, dq, ds = ctx.saved_tensors
        k, (tg, tu, td) = ctx.use_kernel, ctx.dtypes
        need_x, need_g, need_u, need_d = ctx.needs_input_grad[:4]
        dwd = _weight_grad(dy, h_q, sh, k, td) if need_d else None
        if not (need_x or need_g or need_u):
            return None, None, None, dwd, None, None
        dg, du = _silu_mul_grad(_input_grad(dy, dq, ds, k), (kq, ks), k)
        dwg = _weight_grad(dg, x_q, sx, k, tg) if need_g else None
        dwu = _weight_grad(du, x_q, sx, k, tu) if need_u else None
        # (each product rounded to x's type, then their sum: as autograd adds what two layers give)
        dx = _input_grad(dg, gq, gs, k).add_(_input_grad(du, uq, us, k)) if need_x else None
        return dx, dwg, dwu, dwd, None, None


class Int8Linear(nn.Module):
    """A linear layer for training with INT8 products: the parameters keep their dtype and are quantized at every
    forward; x may be float32, float16 or bfloat16, and y has its dtype."""

    def __init__(self, linear: nn.Linear, use_kernel: bool = True):
        super().__init__()
        copy = lambda p: None if p is None else nn.Parameter(p.detach().clone(), requires_grad=p.requires_grad)
        self.weight, self.bias = copy(linear.weight), copy(linear.bias)
        self.use_kernel = use_kernel

    @property
    def out_features(self) -> int:
        return self.weight.shape[0]

    @property
    def in_features(self) -> int:
        return self.weight.shape[1]

    def forward(self, x):
        y = _Int8LinearFn.apply(x.reshape(-1, x.shape[-1]), self.weight, self.bias, self.use_kernel)
        return y.reshape(*x.shape[:-1], self.weight.shape[0])


class Int8SwiGLU(nn.Module):
    """w_down(silu(w_gate(x)) * w_up(x)) for training with INT8 products and 8-bit activations, under the
    parameter names of the reference's SwiGLU (train/model.py:127-135). No biases. With other layers put in their places
    (serve.quantize.quantize_model's), or hooks on one of its own, it calls the three one after another."""

    def __init__(self, w_gate: nn.Linear, w_up: nn.Linear, w_down: nn.Linear, use_kernel: bool = True):
        super().__init__()
        if any(m.bias is not None for m in (w_gate, w_up, w_down)):
            raise ValueError("Int8SwiGLU: projections with biases")
        own = lambda m: m if isinstance(m, Int8Linear) else Int8Linear(m, use_kernel)
        self.w_gate, self.w_up, self.w_down = own(w_gate), own(w_up), own(w_down)
        self.use_kernel = use_kernel

    def forward(self, x):
        lins = self.w_gate, self.w_up, self.w_down
        if not all(isinstance(m, Int8Linear) for m in lins) or has_hooks(*lins):
            return self.w_down(nn.functional.silu(self.w_gate(x)) * self.w_up(x))
        y = _Int8SwiGLUFn.apply(x.reshape(-1, x.shape[-1]), self.w_gate.weight, self.w_up.weight, self.w_down.weight,
                                self.use_kernel, torch.is_grad_enabled())
        return y.reshape(*x.shape[:-1], self.w_down.weight.shape[0])


def convert_linears_to_int8(model: nn.Module, use_kernel: bool = True) -> nn.Module:
    """A copy of the model whose attention projections (wq/wk/wv/wo) are Int8Linear and whose SwiGLU MLPs (modules with
    w_gate/w_up/w_down) are Int8SwiGLU; embeddings, head, router and norms stay as they are. Modules are recognised by their slot names, as
    train.fp8.convert_linears_to_fp8 does, and an MLP with biases or that computes something else (serve.quantize.computes_swiglu) keeps its forward,
    over three Int8Linear. The state dict keeps its names, and what is shared in the model is in the copy."""
    import copy
    model = copy.deepcopy(model)
    made = {}  # id of a layer or MLP of the copy -> itself and what takes its place, the same in all of its places

    def once(m, make):
        if id(m) not in made:
            made[id(m)] = m, make().train(m.training)
        return made[id(m)][1]

    def linear(lin):
        def make():
            new = Int8Linear(lin, use_kernel)
            new.weight, new.bias = lin.weight, lin.bias  # (the copy's own, which others may share)
            return new
        return once(lin, make)

    def linears(m, names):
        lins = [getattr(m, n, None) for n in names]
        return lins if all(isinstance(lin, nn.Linear) for lin in lins) else None

    def fused(m):
        lins = linears(m, _MLP)
        if lins is None:
            return m
        if all(lin.bias is None for lin in lins) and computes_swiglu(m):
            return once(m, lambda: Int8SwiGLU(*(linear(lin) for lin in lins), use_kernel=use_kernel))
        for n, lin in zip(_MLP, lins):
            setattr(m, n, linear(lin))
        return m

    for m in list(model.modules()):
        for n, lin in zip(_ATTN, linears(m, _ATTN) or ()):
            setattr(m, n, linear(lin))
        for name, child in list(m._modules.items()):  # (named_children names a child that stands twice once)
            if child is not None and (new := fused(child)) is not child:
                setattr(m, name, new)
    return fused(model)
