"""Weight-only quantization: INT8 (per-row symmetric) and INT4 (group-wise).

Same functions, classes and buffer layouts as the reference's serve/quantize.py
(:18-129), so a serving engine built on nn.Linear slots runs unchanged:

INT8: scale[n] = max|w[n]| / 127 (floored at 1e-8); w_q = round-half-even(w / scale)
      clamped to [-127, 127].
INT4: per group of `group_size` along K, scale = max|w_group| / 7 (floored at
      1e-8); q = clamp(round(w / scale), -8, 7) + 8, two nibbles per byte with
      even k in the low nibble.

Quantization is load-time work. On HIP tensors it runs the gfx950 quantizer
kernels (bit-exact: IEEE division, ties to even); on host tensors (a model
quantized before it is moved to the GPU, as the reference's CLI does) it runs
the reference's host op sequence, which is the definition the kernels match.
QuantLinear(use_kernel=True) runs the fused HIP GEMMs of kernels.dequant_matmul;
use_kernel=False keeps the reference's dequantize-then-matmul path.

act_bits=8 (no reference counterpart): the input is quantized too, per token as it comes, and INT8 weights meet it
on the 8-bit matrix cores (kernels.int8_act), at about twice the 16-bit rate for prompts. quantize_model(act_bits=8) also makes
every SwiGLU (computes_swiglu) an Int8SwiGLU, whose product with the down projection's codes is one kernel. Such layers serve: they have
no gradient and refuse inputs that ask for one.

Unlike the reference, this module does not import the model package (the
reference imports train.model only for a type annotation, :15): quantize_model
finds the Linear slots by attribute name.
"""

from __future__ import annotations

import sys

import torch
import torch.nn as nn


def _hip_quantizer():
    import kernels
    from kernels._hip import ld, stream
    return kernels, ld, stream


def quantize_int8(w: torch.Tensor):
    """(w_q int8 [N, K], scale fp32 [N]) -- serve/quantize.py:18-21."""
    if w.device.type != "cuda":
        scale = (w.abs().amax(dim=1) / 127.0).clamp(min=1e-8)
        w_q = torch.round(w / scale[:, None]).clamp(-127, 127).to(torch.int8)
        return w_q, scale
    kernels, ld, stream = _hip_quantizer()
    w32 = w.detach().to(torch.float32)
    if w32.stride(1) != 1:
        w32 = w32.contiguous()
    N, K = w32.shape
    w_q = torch.empty(N, K, dtype=torch.int8, device=w.device)
    scale = torch.empty(N, dtype=torch.float32, device=w.device)
    kernels.check(kernels.lib().mls_quantize_int8(
        w32.data_ptr(), N, K, ld(w32), w_q.data_ptr(), ld(w_q), scale.data_ptr(),
        stream(w.device)), "quantize_int8")
    return w_q, scale


def dequantize_int8(w_q: torch.Tensor, scale: torch.Tensor):
    return w_q.float() * scale[:, None]


def quantize_int4(w: torch.Tensor, group_size: int = 32):
    """(packed uint8 [N, K/2], scale fp32 [N, K/group_size]) -- serve/quantize.py:28-36."""
    N, K = w.shape
    assert K % group_size == 0
    if w.device.type != "cuda" or group_size % 2 or K % 2:
        g = w.reshape(N, K // group_size, group_size)
        scale = (g.abs().amax(dim=2) / 7.0).clamp(min=1e-8)
        q = torch.round(g / scale[:, :, None]).clamp(-8, 7) + 8
        q = q.reshape(N, K).to(torch.uint8)
        packed = (q[:, 0::2] | (q[:, 1::2] << 4)).contiguous()
        return packed, scale
    kernels, ld, stream = _hip_quantizer()
    w32 = w.detach().to(torch.float32)
    if w32.stride(1) != 1:
        w32 = w32.contiguous()
    packed = torch.empty(N, K // 2, dtype=torch.uint8, device=w.device)
    scale = torch.empty(N, K // group_size, dtype=torch.float32, device=w.device)
    kernels.check(kernels.lib().mls_quantize_int4(
        w32.data_ptr(), N, K, ld(w32), group_size, packed.data_ptr(), ld(packed),
        scale.data_ptr(), stream(w.device)), "quantize_int4")
    return packed, scale


def dequantize_int4(packed: torch.Tensor, scale: torch.Tensor, group_size: int):
    N = packed.shape[0]
    K = packed.shape[1] * 2
    q = torch.empty(N, K, dtype=torch.uint8, device=packed.device)
    q[:, 0::2] = packed & 0x0F
    q[:, 1::2] = packed >> 4
    w = q.float() - 8.0
    w = w.reshape(N, K // group_size, group_size) * scale.float()[:, :, None]
    return w.reshape(N, K)


def _act_bits(act_bits: int | None, bits: int) -> int | None:
    if act_bits not in (None, 8) or act_bits == 8 and bits != 8:
        raise ValueError(f"act_bits={act_bits} with bits={bits}: activations of 8 bits meet weights of 8, or stay as they are (None)")
    return act_bits


def _no_grad_of(fn: str, *tensors) -> None:
    """The kernels' refusal of inputs that ask for a gradient, for their torch form (whose scales would carry one)."""
    from kernels.paged_kv import no_grad_of
    no_grad_of(fn, *tensors)


class QuantLinear(nn.Module):
    """Drop-in nn.Linear replacement holding quantized weights (serve/quantize.py:50-95).

    use_kernel=True runs the fused gfx950 dequant GEMM; False runs the
    reference path (explicit dequant then matmul), kept for correctness tests
    and host execution. act_bits=8 (with bits=8): x is quantized per token too.
    """

    act_bits: int | None = None

    def __init__(self, linear: nn.Linear, bits: int = 8, group_size: int = 32,
                 use_kernel: bool = True, act_bits: int | None = None):
        super().__init__()
        assert linear.bias is None
        assert bits in (4, 8)
        self.bits, self.group_size, self.use_kernel = bits, group_size, use_kernel
        self.act_bits = _act_bits(act_bits, bits)
        self.out_features, self.in_features = linear.weight.shape
        w = linear.weight.detach().float()
        if bits == 8:
            w_q, scale = quantize_int8(w)
        else:
            w_q, scale = quantize_int4(w, group_size)
        self.register_buffer("w_q", w_q)
        self.register_buffer("scale", scale)

    @classmethod
    def from_quantized(cls, w_q: torch.Tensor, scale: torch.Tensor, bits: int, group_size: int,
                       in_features: int, use_kernel: bool = True, act_bits: int | None = None) -> "QuantLinear":
        """A QuantLinear around buffers that are already quantized (a quantized
        checkpoint): no fp weight, no quantization pass."""
        assert bits in (4, 8)
        self = cls.__new__(cls)
        nn.Module.__init__(self)
        self.bits, self.group_size, self.use_kernel = bits, group_size, use_kernel
        self.act_bits = _act_bits(act_bits, bits)
        self.out_features, self.in_features = w_q.shape[0], in_features
        want = in_features if bits == 8 else in_features // 2
        if w_q.dim() != 2 or w_q.shape[1] != want:
            raise ValueError(f"QuantLinear.from_quantized: w_q {tuple(w_q.shape)} does not hold "
                             f"{in_features} int{bits} columns")
        self.register_buffer("w_q", w_q)
        self.register_buffer("scale", scale)
        return self

    def dequant(self) -> torch.Tensor:
        if self.bits == 8:
            return dequantize_int8(self.w_q, self.scale)
        return dequantize_int4(self.w_q, self.scale, self.group_size)

    def weight_bytes(self) -> int:
        return self.w_q.numel() * self.w_q.element_size() + \
            self.scale.numel() * self.scale.element_size()

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        shape = x.shape
        flat = x.reshape(-1, self.in_features)
        if self.act_bits == 8:
            if self.use_kernel:
                from kernels.int8_act import int8_dynamic_matmul
                y = int8_dynamic_matmul(flat, self.w_q, self.scale)
            else:
                _no_grad_of("QuantLinear(act_bits=8)", flat)
                y = self.matmul_codes(*quantize_int8(flat.float()), flat.dtype)
        elif self.use_kernel:
            from kernels.dequant_matmul import int4_matmul, int8_matmul
            if self.bits == 8:
                y = int8_matmul(flat, self.w_q, self.scale)
            else:
                y = int4_matmul(flat, self.w_q, self.scale, self.group_size)
        else:
            y = flat @ self.dequant().to(flat.dtype).t()
        return y.reshape(*shape[:-1], self.out_features)

    def matmul_codes(self, x_q: torch.Tensor, sx: torch.Tensor, out_dtype: torch.dtype) -> torch.Tensor:
        """forward of an input that is quantized per token already: codes [M, K], scales [M]."""
        if self.use_kernel:
            from kernels.int8_act import int8_scaled_matmul
            return int8_scaled_matmul(x_q, sx, self.w_q, self.scale, out_dtype=out_dtype)
        _no_grad_of("QuantLinear.matmul_codes", sx, self.scale)
        return ((x_q.double() @ self.w_q.double().t()) * self.scale.double() * sx.double()[:, None]).to(out_dtype)


def has_hooks(*modules: nn.Module) -> bool:
    """Whether calling one of these runs more than its forward."""
    return any(m._forward_hooks or m._forward_pre_hooks or m._backward_hooks or m._backward_pre_hooks for m in modules)


class Int8SwiGLU(nn.Module):
    """w_down(silu(w_gate(x)) * w_up(x)) of three QuantLinear(act_bits=8), under the names that the
    reference's SwiGLU gives them (train/model.py:127-135): x is quantized once for gate and up, and the product
    once more, in fp32, on its way to w_down. The three are not called themselves, unless one has hooks: then each is, and the
    product is rounded to x's dtype in between."""

    def __init__(self, w_gate: QuantLinear, w_up: QuantLinear, w_down: QuantLinear):
        super().__init__()
        for m in (w_gate, w_up, w_down):
            if not (isinstance(m, QuantLinear) and m.act_bits == 8):
                raise ValueError("Int8SwiGLU needs three QuantLinear with act_bits=8")
        self.w_gate, self.w_up, self.w_down = w_gate, w_up, w_down

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        if has_hooks(self.w_gate, self.w_up, self.w_down):
            g, u = self.w_gate(x).float(), self.w_up(x).float()
            return self.w_down((g * torch.sigmoid(g) * u).to(x.dtype))
        flat = x.reshape(-1, x.shape[-1])
        if not self.w_gate.use_kernel:
            _no_grad_of("Int8SwiGLU", flat)
            xq = quantize_int8(flat.float())
            g, u = (m.matmul_codes(*xq, flat.dtype).float() for m in (self.w_gate, self.w_up))
            h = quantize_int8(g * torch.sigmoid(g) * u)
        else:
            from kernels.int8_act import int8_dynamic_matmul, quantize_rows, silu_mul_quantize
            # (up to 16 rows both products take x: where they quantize it on the way that is a launch less, and where they do not, from 5 rows
            # of 4096 -> 11008, one more)
            if flat.shape[0] <= 16:
                g, u = (int8_dynamic_matmul(flat, m.w_q, m.scale) for m in (self.w_gate, self.w_up))
            else:
                xq = quantize_rows(flat)
                g, u = (m.matmul_codes(*xq, flat.dtype) for m in (self.w_gate, self.w_up))
            h = silu_mul_quantize(g, u)
        return self.w_down.matmul_codes(*h, flat.dtype).reshape(*x.shape[:-1], self.w_down.out_features)


_ATTN_SLOTS = ("wq", "wk", "wv", "wo")
_MLP_SLOTS = ("w_gate", "w_up", "w_down")


def computes_swiglu(m: nn.Module) -> bool:
    """Whether a module with a SwiGLU's slots computes w_down(silu(w_gate(x)) * w_up(x)) and nothing else, so that one that does may take
    its place. It is asked, not its name: its forward runs in both modes on small numbers in 64 bits, with layers of the probe's in the slots.
    A module with state of its own or hooks is not replaced, one without a forward says nothing against it."""
    import copy
    others = [c for n, c in m.named_children() if n not in _MLP_SLOTS]
    if has_hooks(m) or m._parameters or m._buffers or any(c.state_dict() for c in others):
        return False
    if type(m).forward is nn.Module.forward and "forward" not in m.__dict__:
        return True
    D, H, kw = 8, 64, dict(dtype=torch.float64, device="cpu")
    g = torch.Generator("cpu").manual_seed(0)
    with torch.no_grad(), torch.random.fork_rng(devices=[]):
        slots = {n: nn.Linear(a, b, bias=False, **kw) for n, a, b in zip(_MLP_SLOTS, (D, D, H), (H, H, D))}
        for lin in slots.values():
            lin.weight.copy_(torch.randn(lin.weight.shape, generator=g, **kw))
        x = 2 * torch.randn(64, D, generator=g, **kw)
        want = slots["w_down"](nn.functional.silu(slots["w_gate"](x)) * slots["w_up"](x))
        try:
            probe = copy.copy(m)
            probe._modules = {n: slots[n] if n in slots else copy.deepcopy(c) for n, c in m._modules.items()}
            # (1e-5 of the norm: a forward may go through fp32, and one value dropped of the 4096 between the layers is 1e-2)
            return all(float((probe.train(mode)(x) - want).norm()) <= 1e-5 * float(want.norm()) for mode in (True, False))
        except Exception:  # (another shape, type or argument: not this function)
            return False


def _fuse_int8_mlps(model: nn.Module) -> None:
    """Every SwiGLU of the blocks whose three projections have act_bits=8 becomes an Int8SwiGLU."""
    def fused(m):
        lins = [getattr(m, n, None) for n in _MLP_SLOTS]
        ok = not isinstance(m, Int8SwiGLU) and all(isinstance(q, QuantLinear) and q.act_bits == 8 for q in lins) and computes_swiglu(m)
        return Int8SwiGLU(*lins).train(m.training) if ok else m
    for blk in getattr(model, "blocks", []):
        if getattr(blk, "is_moe", False):
            for i, m in enumerate(blk.mlp.experts):
                blk.mlp.experts[i] = fused(m)
        elif hasattr(blk, "mlp"):
            blk.mlp = fused(blk.mlp)


def quantize_model(model: nn.Module, bits: int = 8, group_size: int = 32,
                   use_kernel: bool = True, act_bits: int | None = None) -> nn.Module:
    """Replace all block linears with QuantLinear (router/embed/head stay fp)
    (serve/quantize.py:98-115). Walks model.blocks; each block's .attn holds
    wq/wk/wv/wo and its .mlp holds w_gate/w_up/w_down, or, when blk.is_moe,
    .mlp.experts is a list of such MLPs. act_bits=8 (with bits=8): their inputs are
    quantized per token too, and the MLPs that compute a SwiGLU become Int8SwiGLU."""
    import copy
    _act_bits(act_bits, bits)
    model = copy.deepcopy(model)
    for blk in model.blocks:
        a = blk.attn
        for name in _ATTN_SLOTS:
            setattr(a, name, QuantLinear(getattr(a, name), bits, group_size, use_kernel, act_bits))
        mods = blk.mlp.experts if getattr(blk, "is_moe", False) else [blk.mlp]
        for m in mods:
            for name in _MLP_SLOTS:
                setattr(m, name, QuantLinear(getattr(m, name), bits, group_size, use_kernel, act_bits))
        if getattr(blk, "is_moe", False):
            stacked_int4_experts(mods)
    if act_bits is not None:
        _fuse_int8_mlps(model)
    return model


def _expert_slots_ok(experts) -> bool:
    """True when every expert is a SwiGLU MLP (w_down(silu(w_gate(x)) * w_up(x)),
    train/model.py:127-135) whose three projections are INT4 QuantLinear running the
    HIP kernels, with one shape, group size, scale dtype and device across experts, and
    shapes the grouped MFMA kernels take (K % 64 == 0, group % 32 == 0)."""
    if len(experts) == 0:
        return False
    ref = None
    for m in experts:
        lins = [getattr(m, n, None) for n in _MLP_SLOTS]
        if not all(isinstance(q, QuantLinear) and q.bits == 4 and q.use_kernel for q in lins):
            return False
        sig = tuple((tuple(q.w_q.shape), tuple(q.scale.shape), q.scale.dtype, q.group_size, q.w_q.device)
                    for q in lins)
        if ref is None:
            ref = sig
        elif sig != ref:
            return False
    g, u, d = ref
    D, H, group, dev = g[0][1] * 2, g[0][0], g[3], g[4]
    return (dev.type == "cuda" and u == g and d[0] == (D, H // 2) and group % 32 == 0
            and D % 64 == 0 and H % 64 == 0 and g[2] in (torch.float32, torch.float16))


def stacked_int4_experts(experts):
    """Stacked INT4 buffers of a list of SwiGLU experts, for the grouped kernels of
    kernels.moe_grouped: {"w_gate": (packed [E, H, D/2], scale [E, H, D/group]),
    "w_up": (...), "w_down": (packed [E, D, H/2], scale [E, D, H/group]),
    "group_size": g}, or None when the experts do not qualify (_expert_slots_ok).

    The stack is built once: each slot's buffers are copied into one [E, ...] tensor
    and every expert's QuantLinear buffers are re-pointed at views of it, so the
    per-expert modules and the stacked tensors share memory. Later calls only check
    that the buffers are still those views (they are not after .to() or a
    load_state_dict that replaced them) and rebuild when they are not."""
    if not _expert_slots_ok(experts):
        return None
    first = experts[0]
    st = first.__dict__.get("_int4_stack")
    if st is not None and len(st["experts"]) == len(experts) and all(
            a is b for a, b in zip(st["experts"], experts)):
        ok = True
        for name in _MLP_SLOTS:
            wq, sc = st[name]
            for e, m in enumerate(experts):
                q = getattr(m, name)
                if q.w_q.data_ptr() != wq[e].data_ptr() or q.scale.data_ptr() != sc[e].data_ptr():
                    ok = False
                    break
            if not ok:
                break
        if ok:
            return st
    st = {"experts": list(experts), "group_size": first.w_gate.group_size}
    with torch.no_grad():
        for name in _MLP_SLOTS:
            lins = [getattr(m, name) for m in experts]
            wq = torch.stack([q.w_q for q in lins]).contiguous()
            sc = torch.stack([q.scale for q in lins]).contiguous()
            for e, q in enumerate(lins):
                q.w_q = wq[e]
                q.scale = sc[e]
            st[name] = (wq, sc)
    first.__dict__["_int4_stack"] = st
    return st


def model_weight_bytes(model: nn.Module) -> int:
    """Bytes of QuantLinear buffers plus every distinct parameter (serve/quantize.py:118-129)."""
    total = 0
    seen = set()
    for m in model.modules():
        if isinstance(m, QuantLinear):
            total += m.weight_bytes()
    for p in model.parameters():
        if id(p) in seen:
            continue
        seen.add(id(p))
        total += p.numel() * p.element_size()
    return total


# ------------------------------------------------------------------ quantized checkpoints
#
# The reference saves the fp state dict and quantizes again at every load
# (serve/api.py:47, 79-81). A quantized checkpoint stores the QuantLinear buffers
# themselves (w_q, scale: serve/quantize.py:68-73) next to the model's fp parameters,
# in a safetensors file (plain tensors + a string header; loading executes nothing),
# so a load is a copy to the device and quantization runs once, on the GPU.
#
# Header ("__metadata__"): format = "mls-quantized", version = "1", and per quantized
# module "q:<module name>" = "<bits>,<group_size>,<in_features>", and "a:<module name>" = "8" where its
# input is quantized too. Tensors: the model's
# state dict (the QuantLinear buffers under their state-dict names, every other
# parameter and buffer as stored), each saved as its own contiguous copy.

QCKPT_FORMAT, QCKPT_VERSION = "mls-quantized", "1"


def save_quantized(model: nn.Module, path, extra_metadata: dict | None = None) -> None:
    """Write a model whose linears are QuantLinear (quantize_model's output) to a
    quantized safetensors checkpoint at `path`."""
    from safetensors.torch import save_file
    meta = {"format": QCKPT_FORMAT, "version": QCKPT_VERSION}
    for name, m in model.named_modules():
        if isinstance(m, QuantLinear):
            meta[f"q:{name}"] = f"{m.bits},{m.group_size},{m.in_features}"
            if m.act_bits is not None:
                meta[f"a:{name}"] = str(m.act_bits)
    if len(meta) == 2:
        raise ValueError("save_quantized: the model holds no QuantLinear (run quantize_model first)")
    for k, v in (extra_metadata or {}).items():
        if k in meta or k.startswith(("q:", "a:")):
            raise ValueError(f"save_quantized: metadata key {k!r} is reserved")
        meta[k] = str(v)
    tensors = {k: v.detach().contiguous().clone() for k, v in model.state_dict().items()}
    save_file(tensors, str(path), metadata=meta)


def read_quantized_metadata(path) -> dict:
    """The string header of a quantized checkpoint (format, version, modules, extras)."""
    from safetensors import safe_open
    with safe_open(str(path), framework="pt") as f:
        meta = dict(f.metadata() or {})
    if meta.get("format") != QCKPT_FORMAT:
        raise ValueError(f"{path}: not a quantized checkpoint (format {meta.get('format')!r})")
    if meta.get("version") != QCKPT_VERSION:
        raise ValueError(f"{path}: quantized checkpoint version {meta.get('version')!r}, "
                         f"this build reads {QCKPT_VERSION!r}")
    return meta


def _set_submodule(model: nn.Module, name: str, mod: nn.Module) -> None:
    parent, _, leaf = name.rpartition(".")
    setattr(model.get_submodule(parent) if parent else model, leaf, mod)


def load_quantized(model: nn.Module, path, device=None, use_kernel: bool = True) -> nn.Module:
    """Load a quantized checkpoint into `model` (the fp architecture, e.g. a freshly
    built Transformer, or one converted by train.int8; it is modified in place and returned): every module the header
    lists becomes a QuantLinear holding the stored buffers, then the remaining
    parameters load as a state dict (strict: missing or unexpected keys raise). With
    `device`, tensors are read straight onto it. MoE experts are stacked for the
    grouped kernels as quantize_model does."""
    from safetensors.torch import load_file
    meta = read_quantized_metadata(path)
    dev = torch.device(device) if device is not None else None
    # (a model that holds an Int8Linear has imported its module)
    linears = nn.Linear, QuantLinear, getattr(sys.modules.get("train.int8"), "Int8Linear", QuantLinear)
    tensors = load_file(str(path), device=str(dev) if dev is not None else "cpu")
    for key, spec in meta.items():
        if not key.startswith("q:"):
            continue
        name = key[2:]
        bits, group, in_features = (int(x) for x in spec.split(","))
        old = model.get_submodule(name)
        if not isinstance(old, linears):
            raise ValueError(f"load_quantized: {name} is a {type(old).__name__}, not a linear layer")
        w_q, scale = tensors.pop(f"{name}.w_q"), tensors.pop(f"{name}.scale")
        out_features = old.out_features
        if w_q.shape[0] != out_features or in_features != old.in_features:
            raise ValueError(f"load_quantized: {name} stores {w_q.shape[0]}x{in_features}, "
                             f"the model has {out_features}x{old.in_features}")
        act = int(meta[f"a:{name}"]) if f"a:{name}" in meta else None
        _set_submodule(model, name, QuantLinear.from_quantized(w_q, scale, bits, group, in_features, use_kernel, act))
    if dev is not None:
        model.to(dev)
    missing, unexpected = model.load_state_dict(tensors, strict=False)
    quant_keys = {k for k in model.state_dict() if k.endswith((".w_q", ".scale"))
                  and isinstance(model.get_submodule(k.rsplit(".", 1)[0]), QuantLinear)}
    missing = [k for k in missing if k not in quant_keys]
    if missing or unexpected:
        raise ValueError(f"load_quantized: missing {missing[:5]}, unexpected {unexpected[:5]}")
    _fuse_int8_mlps(model)
    for blk in getattr(model, "blocks", []):
        if getattr(blk, "is_moe", False):
            stacked_int4_experts(blk.mlp.experts)
    return model
