"""Appending new keys and values to a paged KV cache, rotated by position on the way (gfx950).

The reference's engine writes its cache by torch indexing, a layer and sequence at a time
(serve/kv_cache.py, serve/engine.py:137-144). Here one launch takes the projections' q, k and
v of any mix of prompts, chunks and single tokens, rotates q and k, and scatters K and V
into the pools that kernels.paged_attention reads. The kernel is csrc/paged_kv.hip.
"""

from __future__ import annotations

import struct

import torch

import kernels
from kernels._hip import dt_code, require_hip, stream

_ARGS = struct.Struct("=10Q23q")  # mlsx_paged_append_args


def int32(t: torch.Tensor, name: str, fn: str, shape: tuple) -> torch.Tensor:
    """An index tensor of the given shape (None: any size) as int32 with unit inner stride."""
    if t.dim() != len(shape) or any(w is not None and w != s for w, s in zip(shape, t.shape)):
        raise ValueError(f"{fn}: {name} {tuple(t.shape)}, expected {tuple('any' if w is None else w for w in shape)}")
    if t.dtype != torch.int32:
        if t.dtype.is_floating_point or t.dtype.is_complex or t.dtype == torch.bool:
            raise TypeError(f"{fn}: {name} must hold integers, got {t.dtype}")
        t = t.to(torch.int32)
    return t if t.stride(-1) == 1 or t.shape[-1] <= 1 else t.contiguous()


def pools(k_pool: torch.Tensor, v_pool: torch.Tensor, fn: str) -> tuple:
    """Strides of the pools, which are read and written in place: never copied."""
    if k_pool.dim() != 4 or v_pool.shape != k_pool.shape or v_pool.dtype != k_pool.dtype:
        raise ValueError(f"{fn}: pools {tuple(k_pool.shape)} {k_pool.dtype} / {tuple(v_pool.shape)} {v_pool.dtype}: expected "
                         f"two of one shape [num_blocks, kv_heads, block_size, head_dim] and type")
    st = k_pool.stride()
    if v_pool.stride() != st or st[3] != 1 and k_pool.shape[3] > 1:
        raise ValueError(f"{fn}: pools need the same strides, 1 for the last dimension, got {st} / {v_pool.stride()}")
    if k_pool.shape[2] < 1:
        raise ValueError(f"{fn}: blocks of no tokens")
    return st


def no_grad_of(fn: str, *tensors) -> None:
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                raise ValueError(f"{fn} has no gradient: call it under torch.no_grad(), or detach its inputs")


def paged_kv_append(q: torch.Tensor | None, k: torch.Tensor, v: torch.Tensor, k_pool: torch.Tensor, v_pool: torch.Tensor,
                    block_tables: torch.Tensor, context_lens: torch.Tensor, cu_seqlens: torch.Tensor | None = None, *,
                    rope: torch.Tensor | None = None, interleaved: bool = False) -> torch.Tensor | None:
    """Writes k, v [T, Hkv, D] into k_pool / v_pool [num_blocks, Hkv, block_size, D] in place and
    returns q [T, Hq, D] rotated (q itself without rope, None without q).

    Sequence s holds rows cu_seqlens[s] .. cu_seqlens[s + 1] (int32 [n + 1]; None: row s); its last row is
    at position context_lens[s] - 1 (the new tokens counted). A row at position p goes to slot
    p % block_size of block block_tables[s, p // block_size]. Positions outside the table and block ids
    outside the pool store nothing; rows of no sequence store nothing, and their q comes out as zeros.

    rope: float32 [positions, rot], the cosines of a position's rot / 2 angles, then their sines; the
    first rot elements of each head are rotated, in pairs x[j], x[j + rot / 2], or, interleaved, x[2 j],
    x[2 j + 1]. A position outside rope comes out as NaN. All of one type (float32, float16, bfloat16)."""
    fn = "paged_kv_append"
    if k.dim() != 3 or v.shape != k.shape:
        raise ValueError(f"{fn}: k {tuple(k.shape)}, v {tuple(v.shape)}: expected two [tokens, kv_heads, head_dim]")
    T, Hkv, D = k.shape
    kv_sb, kv_sh, kv_st, _ = pools(k_pool, v_pool, fn)
    num_blocks, Hp, block_size, Dp = k_pool.shape
    if (Hp, Dp) != (Hkv, D):
        raise ValueError(f"{fn}: k {tuple(k.shape)}, pools {tuple(k_pool.shape)}: heads or head dims differ")
    if k.dtype != k_pool.dtype or v.dtype != k.dtype or q is not None and q.dtype != k.dtype:
        raise TypeError(f"{fn}: q, k, v and the pools must have one dtype, got {q.dtype if q is not None else None}, {k.dtype}, "
                        f"{v.dtype}, {k_pool.dtype}")
    if q is not None and (q.dim() != 3 or q.shape[0] != T or q.shape[2] != D):
        raise ValueError(f"{fn}: q {tuple(q.shape)} for k {tuple(k.shape)}")
    rot = 0
    if rope is not None:
        if rope.dim() != 2 or rope.dtype != torch.float32:
            raise ValueError(f"{fn}: rope must be float32 [positions, rot], got {rope.dtype} {tuple(rope.shape)}")
        rot = rope.shape[1]
        if rot % 2 or rot > D:
            raise ValueError(f"{fn}: rope rotates {rot} of {D} elements: an even number up to the head dim is needed")
        if rope.stride(1) != 1 or rope.stride(0) < rot:
            rope = rope.contiguous()
    n = context_lens.shape[0] if context_lens.dim() == 1 else -1
    lens = int32(context_lens, "context_lens", fn, (None,))
    tables = int32(block_tables, "block_tables", fn, (n, None))
    cu = None
    if cu_seqlens is not None:
        cu = int32(cu_seqlens, "cu_seqlens", fn, (n + 1,))
    elif n != T:
        raise ValueError(f"{fn}: {T} rows for {n} sequences: without cu_seqlens, each has one")
    no_grad_of(fn, q, k, v, k_pool, v_pool)
    dev = require_hip(fn, *(t for t in (k, v, k_pool, v_pool, tables, lens, q, cu, rope) if t is not None))
    if k.stride(2) != 1 and D > 1:
        k = k.contiguous()
    if v.stride(2) != 1 and D > 1:
        v = v.contiguous()
    turn = q is not None and rot > 0
    out, q_st, q_sh, Hq = q, 0, 0, 0
    if turn:
        if q.stride(2) != 1 and D > 1:
            q = q.contiguous()
        Hq = q.shape[1]
        q_st, q_sh, _ = q.stride()
        out = torch.empty((T, Hq, D), dtype=q.dtype, device=dev)
    k_st, k_sh, _ = k.stride()
    v_st, v_sh, _ = v.stride()
    kernels.check(kernels.lib().mlsx_paged_append(_ARGS.pack(
        q.data_ptr() if turn else 0, k.data_ptr(), v.data_ptr(), k_pool.data_ptr(), v_pool.data_ptr(),
        out.data_ptr() if turn else 0, tables.data_ptr(), lens.data_ptr(), cu.data_ptr() if cu is not None else 0,
        rope.data_ptr() if rot else 0, dt_code(k.dtype, fn), q_st, q_sh, k_st, k_sh, v_st, v_sh, kv_sb, max(kv_sh, D), max(kv_st, D),
        tables.stride(0), rope.stride(0) if rot else 0, num_blocks, n, T, Hq, Hkv, D, block_size, tables.shape[1],
        rope.shape[0] if rot else 0, rot, interleaved), stream(dev)), fn)
    return out
