"""An attention layer over a paged KV cache: projections, append and attention in one call.

The reference decodes one token a sequence from its cache (serve/engine.py:101-175) and runs
prompts through its training model. PagedAttentionLayer takes any mix of prompts, chunks of them,
drafted tokens and single tokens, and batches that share a prefix:

    layer = PagedAttentionLayer(wq, wk, wv, wo, head_dim=128, rope=rope_table(4096, 128, device="cuda"))
    layer.to_int(bits=4, group_size=128)              # the projections as quantized linears
    y = layer(x, k_pool, v_pool, tables, lens, cu)    # prompts: x [tokens, dim], rows cu[s] .. cu[s + 1]
    y = layer(x, k_pool, v_pool, tables, lens)        # a decode step: x [sequences, dim]
    y = layer(x, k_pool, v_pool, tables, lens, prefix=(blocks, 512))  # ... behind 512 tokens cached once

lens counts the new tokens; the caller keeps block tables and lengths, as the reference's BlockManager
does (serve/kv_cache.py). Nothing waits for the GPU, so a decode step can be captured in a graph.
"""

from __future__ import annotations

import torch
import torch.nn as nn

from kernels.paged_attention import paged_attention, shared_prefix_attention
from kernels.paged_kv import no_grad_of, paged_kv_append
from serve.quantize import QuantLinear


def rope_table(positions: int, rot: int, theta: float = 10000.0, device=None) -> torch.Tensor:
    """float32 [positions, rot]: cosines, then sines, of position * theta^(-2 j / rot), in 64 bits before their rounding."""
    j = torch.arange(rot // 2, dtype=torch.float64)
    angles = torch.arange(positions, dtype=torch.float64)[:, None] * theta ** (-2.0 * j / rot)
    return torch.cat([angles.cos(), angles.sin()], 1).float().to(device)


class PagedAttentionLayer(nn.Module):
    """y = wo(attention(wq x, cache with wk x and wv x added)); the options are paged_attention's."""

    def __init__(self, wq: nn.Module, wk: nn.Module, wv: nn.Module, wo: nn.Module, head_dim: int, *,
                 rope: torch.Tensor | None = None, interleaved: bool = False, scale: float | None = None,
                 softcap: float = 0.0, slopes: torch.Tensor | None = None, window: int = 0):
        super().__init__()
        for name, m in (("wq", wq), ("wk", wk), ("wv", wv)):
            if m.out_features % head_dim:
                raise ValueError(f"PagedAttentionLayer: {name} makes {m.out_features} features, no multiple of {head_dim}")
        if wk.out_features != wv.out_features or wo.in_features != wq.out_features:
            raise ValueError(f"PagedAttentionLayer: wk / wv make {wk.out_features} / {wv.out_features} features, wo takes "
                             f"{wo.in_features} of wq's {wq.out_features}")
        self.wq, self.wk, self.wv, self.wo = wq, wk, wv, wo
        self.head_dim, self.interleaved = head_dim, interleaved
        self.options = dict(scale=scale, softcap=softcap, window=window)
        self.register_buffer("rope", rope, persistent=False)
        self.register_buffer("slopes", slopes, persistent=False)

    def _apply(self, fn, recurse=True):
        """Moves the tables with the module, but leaves them float32 under .half() and the like."""
        keep = self.rope, self.slopes
        super()._apply(fn, recurse)
        self.rope, self.slopes = (t if t is None else to.to(t.dtype) if t.is_meta else t.to(to.device)
                                  for t, to in zip(keep, (self.rope, self.slopes)))
        return self

    def to_int(self, bits: int = 8, group_size: int = 32) -> "PagedAttentionLayer":
        """Replaces the projections by quantized ones (serve/quantize.py:98-115 for one layer)."""
        for name in ("wq", "wk", "wv", "wo"):
            setattr(self, name, QuantLinear(getattr(self, name), bits, group_size))
        return self

    def forward(self, x: torch.Tensor, k_pool: torch.Tensor, v_pool: torch.Tensor, block_tables: torch.Tensor,
                context_lens: torch.Tensor, cu_seqlens: torch.Tensor | None = None, *, max_new: int | None = None,
                prefix_lens: torch.Tensor | None = None, prefix: tuple[torch.Tensor, int] | None = None) -> torch.Tensor:
        """prefix: (its blocks, its tokens), cached once for all sequences of a decode step; block_tables and
        context_lens then hold the tokens after it. For serving: the parameters get no gradient, and inputs that ask
        for one are refused."""
        no_grad_of("PagedAttentionLayer", x, k_pool, v_pool)
        with torch.no_grad():
            return self._forward(x, k_pool, v_pool, block_tables, context_lens, cu_seqlens, max_new, prefix_lens, prefix)

    def _forward(self, x, k_pool, v_pool, block_tables, context_lens, cu_seqlens, max_new, prefix_lens, prefix):
        q, k, v = (w(x).unflatten(-1, (-1, self.head_dim)) for w in (self.wq, self.wk, self.wv))
        rope = self.rope
        if prefix is not None:
            if cu_seqlens is not None or prefix_lens is not None:
                raise ValueError("PagedAttentionLayer: a shared prefix goes with one new token a sequence, causal")
            rope = rope[prefix[1]:] if rope is not None else None
        q = paged_kv_append(q, k, v, k_pool, v_pool, block_tables, context_lens, cu_seqlens, rope=rope, interleaved=self.interleaved)
        if prefix is not None:
            y = shared_prefix_attention(q, k_pool, v_pool, *prefix, block_tables, context_lens, slopes=self.slopes, **self.options)
        else:
            y = paged_attention(q, k_pool, v_pool, block_tables, context_lens, cu_seqlens, max_new=max_new, slopes=self.slopes,
                                prefix_lens=prefix_lens, **self.options)
        return self.wo(y.flatten(-2))
