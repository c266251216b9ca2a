"""The operators on 8-bit activations as measurable cases.

Six kinds, each through a public entry point of kernels.int8_act:

  linear   int8_dynamic_matmul: a linear layer that quantizes its input per token and multiplies
           the codes with INT8 weights
  product  int8_scaled_matmul: the same product from codes that are there already
  down     silu_mul_quantize, then int8_scaled_matmul: the second half of a SwiGLU MLP, served
  act_bwd  silu_mul_backward: the gradients of gate and up from their 8-bit checkpoint
  dw       int8_weight_grad: a weight's gradient from an input that was kept in 8 bits
  step     the second half of a SwiGLU MLP in training: silu_mul_quantize with its checkpoint, the
           product, and both gradients from what was kept

A case is a dict of plain values; listed() names the fixed ones, draw(rng) makes more of the
same ranges. With own = False, run() computes the same results in elementary torch operations,
in 32 bits.
"""

from __future__ import annotations

import math
import sys
from pathlib import Path

import torch

_PKG = str(Path(__file__).resolve().parent.parent / "mini-llm-stack_amd")

own = False

_DT = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
_BYTES = {"fp32": 4, "fp16": 2, "bf16": 2}
GROUP = 128  # columns that share a scale in a checkpoint


def listed():
    return [
        # The smallest call: one sequence decoding through an attention projection (latency counts).
        {"name": "linear_bf16_r1", "kind": "linear", "dtype": "bf16", "rows": 1, "k": 4096, "n": 4096, "bias": False},
        # A batch of 16 sequences decoding through an up projection with a bias.
        {"name": "linear_fp16_r16_bias", "kind": "linear", "dtype": "fp16", "rows": 16, "k": 4096, "n": 11008, "bias": True},
        # A prompt through the fp32 engine.
        {"name": "linear_fp32_r200", "kind": "linear", "dtype": "fp32", "rows": 200, "k": 2048, "n": 5632, "bias": False},
        # A ragged chunk of a prompt through a down projection.
        {"name": "linear_bf16_r333", "kind": "linear", "dtype": "bf16", "rows": 333, "k": 11008, "n": 4096, "bias": False},
        # The largest: a long prefill through a wide layer, its input quantized before.
        {"name": "product_bf16_r4096", "kind": "product", "dtype": "bf16", "rows": 4096, "k": 8192, "n": 8192, "bias": False},
        # Odd sizes: a head for 1001 labels on 77 pooled rows.
        {"name": "product_fp16_r77_odd", "kind": "product", "dtype": "fp16", "rows": 77, "k": 777, "n": 1001, "bias": True},
        # A SwiGLU MLP's second half at one token.
        {"name": "down_bf16_r1", "kind": "down", "dtype": "bf16", "rows": 1, "k": 11008, "n": 4096},
        # The backward of the activation on a batch of four sequences of 1024 tokens.
        {"name": "act_bwd_bf16_r4096", "kind": "act_bwd", "dtype": "bf16", "rows": 4096, "k": 11008},
        # A small fp32 training run: 100 tokens, an odd width.
        {"name": "act_bwd_fp32_r100", "kind": "act_bwd", "dtype": "fp32", "rows": 100, "k": 1365},
        # The gradient of an up projection on three sequences of 700 tokens.
        {"name": "dw_bf16_r2100", "kind": "dw", "dtype": "bf16", "rows": 2100, "k": 4096, "n": 11008},
        # Quantization-aware training in fp32.
        {"name": "dw_fp32_r1000", "kind": "dw", "dtype": "fp32", "rows": 1000, "k": 1024, "n": 2048},
        # A training step of a SwiGLU MLP's second half.
        {"name": "step_bf16_r2048", "kind": "step", "dtype": "bf16", "rows": 2048, "k": 5632, "n": 2048},
    ]


def _log(rng, lo, hi, step=1):
    """A multiple of `step` in [lo, hi], spread evenly over the logarithm."""
    v = math.exp(rng.uniform(math.log(lo), math.log(hi)))
    return min(hi // step * step, max(-(-lo // step) * step, int(round(v / step)) * step))


def draw(rng):
    kind = rng.choice(["linear", "linear", "linear", "product", "down", "act_bwd", "dw", "dw", "step"])
    wide = {"linear": ["bf16", "bf16", "fp16", "fp32"], "down": ["bf16", "fp16"], "step": ["bf16", "fp16"]}
    c = {"kind": kind, "dtype": rng.choice(wide.get(kind, ["bf16", "fp16", "fp32"]))}
    step = rng.choice([1, 8, 16, 64, 128, 128])
    if kind == "act_bwd":
        c["rows"], c["k"] = _log(rng, 16, 4096), _log(rng, 256, 11008, step)
        return c
    c["k"], c["n"] = _log(rng, 256, 11008, step), _log(rng, 256, 11008, step)
    if kind in ("linear", "product", "down"):
        c["rows"] = _log(rng, 1, 4096)
        if kind != "down":
            c["bias"] = rng.choice([False, True])
    else:
        c["rows"] = _log(rng, 64, 2048)
    return c


# ---------------------------------------------------------------- inputs, from the seed alone

def _codes_of(x):
    """Codes and scales of the rows of fp32 x, as a checkpoint or a weight holds them."""
    s = (x.abs().amax(-1, keepdim=True) / torch.full((), 127.0, device=x.device)).clamp_min(1e-8)
    return torch.round(x / s).clamp_(-127, 127).to(torch.int8), s.squeeze(-1)


def prepare(case, seed):
    c, dt, rows, k = case, _DT[case["dtype"]], case["rows"], case["k"]
    g = torch.Generator(device="cuda").manual_seed(int(seed))

    def randn(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    def hidden(*shape):
        """Activations: every token of its own size, one feature in 64 well above the others."""
        x = randn(*shape)
        return x * torch.exp(0.5 * randn(shape[0], 1)) * torch.where(torch.rand(shape[1], generator=g, device="cuda") < 1 / 64, 6.0, 1.0)

    st = {"case": dict(c)}
    if c["kind"] != "act_bwd":
        w = randn(c["n"], k) * 0.02
        st["w_q"], st["w_s"] = _codes_of(w)
        st["bias"] = (0.1 * randn(c["n"])).to(dt) if c.get("bias") else None
    if c["kind"] == "linear":
        st["x"] = hidden(rows, k).to(dt)
    elif c["kind"] in ("product", "dw"):
        st["x_q"], st["x_s"] = _codes_of(hidden(rows, k).to(dt).float())
    else:
        st["gate"], st["up"] = (2 * randn(rows, k)).to(dt), hidden(rows, k).to(dt)
    if c["kind"] in ("act_bwd", "step"):
        st["dh"] = (1e-3 * randn(rows, k)).to(dt)
    if c["kind"] in ("dw", "step"):
        st["dy"] = (1e-3 * randn(rows, c["n"])).to(dt)
    if c["kind"] == "act_bwd":
        wide = -(-k // GROUP)
        both = torch.zeros(2, rows, wide * GROUP, device="cuda")
        both[0, :, :k], both[1, :, :k] = st.pop("gate"), st.pop("up")
        q, st["kept_s"] = _codes_of(both.reshape(2, rows, wide, GROUP))
        st["kept_q"] = q.reshape(2, rows, wide * GROUP)[..., :k].contiguous()
    return st


# ---------------------------------------------------------------- one pass

def run(state):
    c = state["case"]
    if not own:
        return _PLAIN[c["kind"]](state)
    if _PKG not in sys.path:
        sys.path.insert(0, _PKG)
    from kernels import int8_act as a8
    dt = _DT[c["dtype"]]
    if c["kind"] == "linear":
        return a8.int8_dynamic_matmul(state["x"], state["w_q"], state["w_s"], state["bias"])
    if c["kind"] == "product":
        return a8.int8_scaled_matmul(state["x_q"], state["x_s"], state["w_q"], state["w_s"], state["bias"], out_dtype=dt)
    if c["kind"] == "down":
        h_q, h_s = a8.silu_mul_quantize(state["gate"], state["up"])
        return a8.int8_scaled_matmul(h_q, h_s, state["w_q"], state["w_s"], out_dtype=dt)
    if c["kind"] == "act_bwd":
        return a8.silu_mul_backward(state["dh"], (state["kept_q"], state["kept_s"]))
    if c["kind"] == "dw":
        return a8.int8_weight_grad(state["dy"], state["x_q"], state["x_s"])
    h_q, h_s, kept = a8.silu_mul_quantize(state["gate"], state["up"], checkpoint=True)
    y = a8.int8_scaled_matmul(h_q, h_s, state["w_q"], state["w_s"], out_dtype=dt)
    dgate, dup = a8.silu_mul_backward(state["dh"], kept)
    return y, dgate, dup, a8.int8_weight_grad(state["dy"], h_q, h_s)


def _rows_8bit(x):
    """Codes (whole numbers in fp32) and scales of the last axis."""
    s = (x.abs().amax(-1, keepdim=True) / torch.full((), 127.0, device=x.device)).clamp_min(1e-8)
    return torch.round(x / s).clamp(-127, 127), s


def _groups_8bit(x):
    """x as its checkpoint gives it back: 8 bits, a scale for every GROUP columns."""
    k = x.shape[1]
    p = torch.nn.functional.pad(x, (0, -k % GROUP)).unflatten(1, (-1, GROUP))
    q, s = _rows_8bit(p)
    return (q * s).flatten(1)[:, :k]


def _product(q, s, state, dtype):
    y = (q @ state["w_q"].float().t()) * state["w_s"] * s
    if state["bias"] is not None:
        y = y + state["bias"].float()
    return y.to(dtype)


def _plain_linear(state):
    q, s = _rows_8bit(state["x"].float())
    return _product(q, s, state, state["x"].dtype)


def _plain_product(state):
    return _product(state["x_q"].float(), state["x_s"][:, None], state, _DT[state["case"]["dtype"]])


def _silu_mul_8bit(gate, up):
    return _rows_8bit(gate / (1 + torch.exp(-gate)) * up)


def _plain_down(state):
    q, s = _silu_mul_8bit(state["gate"].float(), state["up"].float())
    return _product(q, s, state, state["gate"].dtype)


def _silu_mul_grad(dh, gate, up):
    sig = 1 / (1 + torch.exp(-gate))
    d = dh.float()
    return (d * up * sig * (1 + gate * (1 - sig))).to(dh.dtype), (d * gate * sig).to(dh.dtype)


def _plain_act_bwd(state):
    k = state["case"]["k"]
    s = state["kept_s"].repeat_interleave(GROUP, dim=2)[..., :k]
    gate, up = state["kept_q"].float() * s
    return _silu_mul_grad(state["dh"], gate, up)


def _plain_dw(state):
    x = state["x_q"].float() * state["x_s"][:, None]
    return (state["dy"].float().t() @ x).to(state["dy"].dtype)


def _plain_step(state):
    gate, up = state["gate"].float(), state["up"].float()
    q, s = _silu_mul_8bit(gate, up)
    y = _product(q, s, state, state["gate"].dtype)
    dgate, dup = _silu_mul_grad(state["dh"], _groups_8bit(gate), _groups_8bit(up))
    return y, dgate, dup, (state["dy"].float().t() @ (q * s)).to(state["dy"].dtype)


_PLAIN = {"linear": _plain_linear, "product": _plain_product, "down": _plain_down, "act_bwd": _plain_act_bwd,
          "dw": _plain_dw, "step": _plain_step}


# ---------------------------------------------------------------- the definition in 64 bits

def exact(case, seed):
    """The operators' definition. A code is the nearest whole number of a quotient rounded to 32 bits and a
    scale a number of 32 bits, which is what the 8-bit forms hold; everything else is in 64 bits."""
    st, c = prepare(case, seed), case
    hundred27 = torch.tensor(127.0, dtype=torch.float32, device="cuda")

    def eight(x):  # x in 64 bits, one scale a row
        big = torch.maximum(x.max(dim=-1).values, -x.min(dim=-1).values).float()
        scale = torch.maximum(big / hundred27, torch.full_like(big, 1e-8))
        return torch.special.round((x.float() / scale.unsqueeze(-1))).double(), scale.double()

    def kept(x):
        parts = [eight(p.contiguous()) for p in x.double().split(GROUP, dim=1)]
        return torch.cat([q * s.unsqueeze(1) for q, s in parts], dim=1)

    def linear(q, s):
        y = torch.mm(q, st["w_q"].double().t()) * torch.outer(s, st["w_s"].double())
        return y if st["bias"] is None else y + st["bias"].double().expand_as(y)

    def grads(gate, up, dh):
        d = dh.double()
        sig = torch.sigmoid(gate)
        slope = sig + gate * sig * torch.sigmoid(-gate)
        return d * slope * up, d * sig * gate

    if c["kind"] == "linear":
        return linear(*eight(st["x"].double()))
    if c["kind"] == "product":
        return linear(st["x_q"].double(), st["x_s"].double())
    if c["kind"] == "dw":
        return torch.mm((st["dy"].double() * st["x_s"].double().unsqueeze(1)).t(), st["x_q"].double())
    if c["kind"] == "act_bwd":
        scale = st["kept_s"].double()[..., torch.arange(c["k"], device="cuda") // GROUP]
        both = st["kept_q"].double() * scale
        return grads(both[0], both[1], st["dh"])
    gate, up = st["gate"].double(), st["up"].double()
    q, s = eight(gate * torch.sigmoid(gate) * up)
    y = linear(q, s)
    if c["kind"] == "down":
        return y
    dgate, dup = grads(kept(gate), kept(up), st["dh"])
    return y, dgate, dup, torch.mm((st["dy"].double() * s.unsqueeze(1)).t(), q)


# ---------------------------------------------------------------- what a pass cannot do without

def work(case):
    c, size, rows, k = case, _BYTES[case["dtype"]], case["rows"], case["k"]
    n = c.get("n", 0)
    scales = 8 * rows * -(-k // GROUP)
    if c["kind"] == "act_bwd":
        return {"bytes": rows * k * (3 * size + 2) + scales, "flops": 12 * rows * k}
    product = 2 * rows * k * n
    if c["kind"] == "dw":
        return {"bytes": rows * n * size + rows * k + 4 * rows + n * k * size, "flops": product}
    weights = n * k + 4 * n + (n * size if c.get("bias") else 0)
    if c["kind"] == "linear":
        return {"bytes": rows * k * size + weights + rows * n * size, "flops": product}
    if c["kind"] == "product":
        return {"bytes": rows * k + 4 * rows + weights + rows * n * size, "flops": product}
    if c["kind"] == "down":
        return {"bytes": 2 * rows * k * size + weights + rows * n * size, "flops": product}
    # gate, up, dh and dy in, y and both gradients out (the checkpoint between them is written and read)
    return {"bytes": rows * k * size * 5 + 4 * rows * k + 2 * scales + rows * n * size * 2 + weights + n * k * size, "flops": 2 * product}
