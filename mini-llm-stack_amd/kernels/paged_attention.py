"""Paged-attention decode over a block-scattered KV cache, on gfx950.

Same function, arguments and result as the reference (kernels/paged_attention.py:
93-118): q [n_seqs, H, D]; k_pool / v_pool [num_blocks, H, block_size, D] (one
(block, head) slab contiguous, K and V with the same strides); block_tables
[n_seqs, max_blocks] int32; context_lens [n_seqs] int32 (the new token already
written and counted); scale defaults to D^-0.5. Returns [n_seqs, H, D] in q's dtype.

The kernel (csrc/paged_attn.hip) walks each sequence's block table and keeps an
online softmax, one wavefront per (sequence, head, piece of the context); contexts are
cut into pieces of one length (128 tokens or more) and merged by a second kernel through a
workspace this wrapper allocates (its size comes from mlsx_paged_attention_workspace). Tokens at or past a sequence's context
length weigh 0; a zero context gives a zero output.

paged_attention and shared_prefix_attention (csrc/paged_gqa.h, csrc/paged_gqa.hip; no reference
counterpart) take any number of new tokens a sequence, several query heads a K/V head, capped
scores, a bias by distance, windows, prefix masks, and batches behind one shared prefix.
"""

from __future__ import annotations

import struct

import torch
from torch.autograd import forward_ad

import kernels
from kernels._hip import _DT, dt_code, require_hip, stream
from kernels.paged_kv import _raw_stream, fresh, int32, no_grad_of, one_device, pools

_ARGS = struct.Struct("=10Q21q2d")  # mlsx_paged_attention_args


def paged_attention_decode(q: torch.Tensor, k_pool: torch.Tensor, v_pool: torch.Tensor,
                           block_tables: torch.Tensor, context_lens: torch.Tensor,
                           scale: float | None = None) -> torch.Tensor:
    dev = require_hip("paged_attention_decode", q, k_pool, v_pool, block_tables, context_lens)
    n_seqs, H, D = q.shape
    num_blocks, Hk, block_size, Dk = k_pool.shape
    if (Hk, Dk) != (H, D) or v_pool.shape != k_pool.shape or v_pool.dtype != k_pool.dtype:
        raise ValueError(f"paged_attention_decode: q {tuple(q.shape)}, pools {tuple(k_pool.shape)} / "
                         f"{tuple(v_pool.shape)} do not match")
    scale = scale if scale is not None else D ** -0.5
    # a fresh dense output whatever q's layout (empty_like would copy q's strides)
    out = torch.empty(n_seqs, H, D, dtype=q.dtype, device=dev)
    if n_seqs == 0:
        return out
    # the library reads q rows with unit inner stride and non-overlapping heads and
    # sequences (q_sh >= D, q_ss >= H*D); any other layout is copied dense first
    # (clone, not contiguous(): a size-1 dimension may keep any stride under contiguous())
    if q.stride(2) != 1 or q.stride(1) < D or q.stride(0) < H * D:
        q = q.clone(memory_format=torch.contiguous_format)
    st = k_pool.stride()
    if (st[3] != 1 or st[2] < D or st[1] < st[2] * block_size or st[0] < st[1] * H
            or v_pool.stride() != st):
        k_pool = k_pool.clone(memory_format=torch.contiguous_format)
        v_pool = v_pool.clone(memory_format=torch.contiguous_format)
    bt = block_tables.to(torch.int32).contiguous()
    ctx = context_lens.to(torch.int32).contiguous()
    if bt.dim() != 2 or bt.shape[0] != n_seqs or ctx.shape != (n_seqs,):
        raise ValueError(f"paged_attention_decode: block_tables {tuple(bt.shape)} / context_lens "
                         f"{tuple(ctx.shape)} for {n_seqs} sequences")
    max_blocks = bt.shape[1]
    L = kernels.lib()
    ws_n = L.mlsx_paged_attention_workspace(n_seqs, H, D, block_size, max_blocks)
    ws = torch.empty(max(ws_n, 1), dtype=torch.float32, device=dev)
    kernels.check(L.mlsx_paged_attention_decode(
        q.data_ptr(), dt_code(q.dtype, "paged_attention_decode q"), q.stride(0), q.stride(1),
        k_pool.data_ptr(), v_pool.data_ptr(), dt_code(k_pool.dtype, "paged_attention_decode pools"),
        k_pool.stride(0), k_pool.stride(1), k_pool.stride(2), num_blocks,
        bt.data_ptr(), bt.stride(0) if n_seqs > 1 else max_blocks, max_blocks, ctx.data_ptr(),
        out.data_ptr(), out.stride(0), out.stride(1), n_seqs, H, D, block_size, float(scale),
        ws.data_ptr(), ws_n, stream(dev)), "paged_attention_decode")
    return out


def _attend(fn, q, k_pool, v_pool, block_tables, context_lens, cu_seqlens, max_new, scale, softcap, slopes, window, prefix_lens,
            prefix_blocks, prefix_len):
    qs, ps, dt, int32_t = q.shape, k_pool.shape, q.dtype, torch.int32
    if len(qs) != 3:
        raise ValueError(f"{fn}: q {tuple(qs)}, expected [tokens, heads, head_dim]")
    T, Hq, D = qs
    kv_sb, kv_sh, kv_st = pools(k_pool, v_pool, fn)
    num_blocks, Hkv, block_size, Dk = ps
    if Dk != D or Hkv < 1 or Hq % Hkv:
        raise ValueError(f"{fn}: q {tuple(qs)}, pools {tuple(ps)}: head dims differ, or query heads are no multiple of K/V heads")
    if k_pool.dtype != dt:
        raise TypeError(f"{fn}: q {dt} and pools {k_pool.dtype} must have one dtype")
    n = context_lens.shape[0] if context_lens.dim() == 1 else -1
    if context_lens.dtype != int32_t or n < 0 or context_lens.stride(0) != 1:
        context_lens = int32(context_lens, "context_lens", fn, (None,))
    ts = block_tables.shape
    if block_tables.dtype != int32_t or len(ts) != 2 or ts[0] != n or block_tables.stride(1) != 1:
        block_tables = int32(block_tables, "block_tables", fn, (n, None))
    cu_at = prefix_at = shared_at = slopes_at = shared_blocks = 0
    if cu_seqlens is not None:
        if cu_seqlens.dtype != int32_t or cu_seqlens.shape != (n + 1,) or cu_seqlens.stride(0) != 1:
            cu_seqlens = int32(cu_seqlens, "cu_seqlens", fn, (n + 1,))
        cu_at = cu_seqlens.data_ptr()
    elif n != T:
        raise ValueError(f"{fn}: {T} rows for {n} sequences: without cu_seqlens, each has one")
    if prefix_lens is not None:
        prefix_lens = int32(prefix_lens, "prefix_lens", fn, (n,))
        prefix_at = prefix_lens.data_ptr()
    if prefix_blocks is not None:
        prefix_blocks = int32(prefix_blocks, "prefix_blocks", fn, (None,))
        shared_blocks = prefix_blocks.shape[0]
        if not 0 <= prefix_len <= shared_blocks * block_size:
            raise ValueError(f"{fn}: a prefix of {prefix_len} tokens in {shared_blocks} blocks of {block_size}")
        shared_at = prefix_blocks.data_ptr() if prefix_len else 0
    if slopes is not None:
        if slopes.shape != (Hq,) or slopes.dtype != torch.float32:
            raise ValueError(f"{fn}: slopes must be float32 [{Hq}], got {slopes.dtype} {tuple(slopes.shape)}")
        slopes = slopes.contiguous()
        slopes_at = slopes.data_ptr()
    if not 0.0 <= softcap < 3e38:
        raise ValueError(f"{fn}: softcap {softcap}: a positive cap, or 0 for none")
    if window < 0 or max_new is not None and max_new < 0:
        raise ValueError(f"{fn}: window {window}, max_new {max_new}: not negative")
    if torch.is_grad_enabled() or forward_ad._current_level >= 0:
        no_grad_of(fn, q, k_pool, v_pool, slopes)
    dev = one_device(fn, q, k_pool, v_pool, block_tables, context_lens, cu_seqlens, prefix_lens, prefix_blocks, slopes)
    q_st, q_sh, inner = q.stride()
    if inner != 1 and D > 1 or q_sh < D and Hq > 1:
        q = q.contiguous()
        q_st, q_sh, _ = q.stride()
    out = fresh(q, qs)
    args = _ARGS.pack(
        q.data_ptr(), k_pool.data_ptr(), v_pool.data_ptr(), block_tables.data_ptr(), context_lens.data_ptr(), cu_at, prefix_at,
        shared_at, slopes_at, out.data_ptr(), _DT[dt] if dt in _DT else dt_code(dt, fn), q_st, q_sh if q_sh > D else D,
        Hq * D, D, kv_sb, kv_sh, kv_st, block_tables.stride(0), num_blocks, n, T, Hkv, Hq // Hkv, D, block_size,
        block_tables.shape[1], window if window < 0x7FFFFFFF else 0x7FFFFFFF, prefix_len, shared_blocks,
        max_new or 0, D ** -0.5 if scale is None else scale, softcap)
    L = kernels.lib()
    need = L.mlsx_paged_attention_ws(args)
    if need:
        ws = q.new_empty(need if dt == torch.float32 else 2 * need)  # (`need` floats)
        rc = L.mlsx_paged_attention(args, ws.data_ptr(), need, _raw_stream(dev))
    else:
        rc = L.mlsx_paged_attention(args, None, 0, _raw_stream(dev))
    if rc:
        kernels.check(rc, fn)
    return out


def paged_attention(q: torch.Tensor, k_pool: torch.Tensor, v_pool: torch.Tensor, block_tables: torch.Tensor,
                    context_lens: torch.Tensor, cu_seqlens: torch.Tensor | None = None, *, max_new: int | None = None,
                    scale: float | None = None, softcap: float = 0.0, slopes: torch.Tensor | None = None, window: int = 0,
                    prefix_lens: torch.Tensor | None = None) -> torch.Tensor:
    """Attention of q [T, Hq, D] over the cached keys and values of each row's sequence; [T, Hq, D].

    k_pool / v_pool [num_blocks, Hkv, block_size, D] of q's type, Hq a multiple of Hkv (query head h reads
    K/V head h // (Hq / Hkv)), any strides with 1 for the last dimension, also 0 for heads, tokens or blocks (an expanded
    view: what they share is read for each). Sequence s holds rows
    cu_seqlens[s] .. cu_seqlens[s + 1] (int32 [n + 1]; None: row s), the newest tokens of its
    context_lens[s] cached ones (written before, as by kernels.paged_kv.paged_kv_append); token j of it is
    slot j % block_size of block block_tables[s, j // block_size]. Offsets rise; where they do not, rows are
    undefined, but no memory besides is touched. max_new: the longest sequence's rows where the
    caller knows them; it only chooses between kernels.

    The row at position p sees token j when j <= p or j < prefix_lens[s] (int32 [n]), and, with a window, when
    p - j < window. A score is scale q.k (scale: D^-0.5), capped softcap tanh(score / softcap), less
    slopes[h] |p - j| (float32 [Hq]). A row that sees nothing (or only scores of -inf) gives zeros, as do rows of no sequence; block ids
    outside the pool hold no tokens, a context longer than its table is cut at the table's end."""
    return _attend("paged_attention", q, k_pool, v_pool, block_tables, context_lens, cu_seqlens, max_new, scale, softcap, slopes,
                   window, prefix_lens, None, 0)


def shared_prefix_attention(q: torch.Tensor, k_pool: torch.Tensor, v_pool: torch.Tensor, prefix_blocks: torch.Tensor,
                            prefix_len: int, block_tables: torch.Tensor, context_lens: torch.Tensor, *,
                            scale: float | None = None, softcap: float = 0.0, slopes: torch.Tensor | None = None,
                            window: int = 0) -> torch.Tensor:
    """A decode step, q [n, Hq, D], of n sequences that all begin with the same prefix_len tokens, cached once
    in the blocks prefix_blocks (int32 [blocks]). block_tables [n, max_blocks] and context_lens [n] hold each
    sequence's own tokens after the prefix, the new one among them, at position prefix_len +
    context_lens[s] - 1. Otherwise as paged_attention over prefix and own tokens, to rounding; the prefix's
    keys and values are read once for all sequences' rows."""
    return _attend("shared_prefix_attention", q, k_pool, v_pool, block_tables, context_lens, None, None, scale, softcap, slopes,
                   window, None, prefix_blocks, prefix_len)
