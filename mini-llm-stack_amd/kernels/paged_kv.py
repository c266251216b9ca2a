"""Appending new keys and values to a paged KV cache, rotated by position on the way (gfx950).

The reference's engine writes its cache by torch indexing, a layer and sequence at a time
(serve/kv_cache.py, serve/engine.py:137-144). Here one launch takes the projections' q, k and
v of any mix of prompts, chunks and single tokens, rotates q and k, and scatters K and V
into the pools that kernels.paged_attention reads. The kernel is csrc/paged_kv.hip.
"""

from __future__ import annotations

import struct

import torch
from torch.autograd import forward_ad

import kernels
from kernels._hip import _DT, dt_code, require_hip

_ARGS = struct.Struct("=10Q23q")  # mlsx_paged_append_args


def int32(t: torch.Tensor, name: str, fn: str, shape: tuple) -> torch.Tensor:
    """An index tensor of the given shape (None: any size) as int32 with unit inner stride; what does not fit becomes the
    nearest value, which is no block id and past every table."""
    if t.dim() != len(shape) or any(w is not None and w != s for w, s in zip(shape, t.shape)):
        raise ValueError(f"{fn}: {name} {tuple(t.shape)}, expected {tuple('any' if w is None else w for w in shape)}")
    if t.dtype != torch.int32:
        if t.dtype.is_floating_point or t.dtype.is_complex or t.dtype == torch.bool:
            raise TypeError(f"{fn}: {name} must hold integers, got {t.dtype}")
        if t.dtype in (torch.int64, torch.uint64, torch.uint32):
            t = t.to(torch.int64).clamp(-2 ** 31, 2 ** 31 - 1)
        t = t.to(torch.int32)
    return t if t.stride(-1) == 1 or t.shape[-1] <= 1 else t.contiguous()


def pools(k_pool: torch.Tensor, v_pool: torch.Tensor, fn: str, write: bool = False) -> tuple:
    """Strides (block, head, token) of the pools, which are read and written in place: never copied. A dimension of size 1
    counts as dense. Heads or tokens of stride 0 (expanded views) can be read, not written."""
    ps = k_pool.shape
    if len(ps) != 4 or v_pool.shape != ps or v_pool.dtype != k_pool.dtype:
        raise ValueError(f"{fn}: pools {tuple(k_pool.shape)} {k_pool.dtype} / {tuple(v_pool.shape)} {v_pool.dtype}: expected "
                         f"two of one shape [num_blocks, kv_heads, block_size, head_dim] and type")
    _, heads, tokens, D = ps
    if tokens < 1:
        raise ValueError(f"{fn}: blocks of no tokens")
    st = k_pool.stride()
    sb, sh, sw, inner = st
    if v_pool.stride() != st or inner != 1 and D > 1:
        raise ValueError(f"{fn}: pools need the same strides, 1 for the last dimension, got {st} / {v_pool.stride()}")
    if heads == 1:
        sh = D
    if tokens == 1:
        sw = D
    if sh < D and sh or sw < D and sw:
        raise ValueError(f"{fn}: pools of strides {st}: heads or tokens overlap within head dims of {D}")
    if write and not (sh and sw and (sh >= sw * (tokens - 1) + D or sw >= sh * (heads - 1) + D)
                      and sb >= sh * (heads - 1) + sw * (tokens - 1) + D):
        end = 1  # (another order of the dimensions, or elements that share memory)
        for step, size in sorted((t, n) for t, n in zip(st, ps) if n > 1):
            if step < end:
                raise ValueError(f"{fn}: pools of shape {tuple(ps)} and strides {st} share memory between elements: they can "
                                 f"be read, not written")
            end += step * (size - 1)
    return sb, sh, sw


_raw_stream = torch._C._cuda_getCurrentRawStream  # (a device index's current stream, as kernels._hip.stream)


def one_device(fn: str, *tensors) -> int:
    """The index of the HIP device that all of these (None: not given) are on."""
    first = tensors[0].get_device()
    if first >= 0:
        for t in tensors:
            if t is not None and t.get_device() != first:
                break
        else:
            return first
    return require_hip(fn, *(t for t in tensors if t is not None)).index


def fresh(like: torch.Tensor, shape: tuple) -> torch.Tensor:
    """A dense uninitialised tensor of `like`'s type and device (empty_like, half the host time, where it is dense)."""
    return torch.empty_like(like) if like.shape == shape and like.is_contiguous() else like.new_empty(shape)


def no_grad_of(fn: str, *tensors) -> None:
    """Refuses tensors that a gradient or a tangent is asked of: the result would silently have none."""
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                raise ValueError(f"{fn} has no gradient: call it under torch.no_grad(), or detach its inputs")
    if forward_ad._current_level >= 0:
        for t in tensors:
            if t is not None and forward_ad.unpack_dual(t).tangent is not None:
                raise ValueError(f"{fn} has no derivative: its inputs must not carry tangents")


def paged_kv_append(q: torch.Tensor | None, k: torch.Tensor, v: torch.Tensor, k_pool: torch.Tensor, v_pool: torch.Tensor,
                    block_tables: torch.Tensor, context_lens: torch.Tensor, cu_seqlens: torch.Tensor | None = None, *,
                    rope: torch.Tensor | None = None, interleaved: bool = False) -> torch.Tensor | None:
    """Writes k, v [T, Hkv, D] into k_pool / v_pool [num_blocks, Hkv, block_size, D] in place and
    returns q [T, Hq, D] rotated (q itself without rope, None without q).

    Sequence s holds rows cu_seqlens[s] .. cu_seqlens[s + 1] (int32 [n + 1]; None: row s); its last row is
    at position context_lens[s] - 1 (the new tokens counted). A row at position p goes to slot
    p % block_size of block block_tables[s, p // block_size]. Positions outside the table and block ids
    outside the pool store nothing; rows of no sequence store nothing, and their rotated q is zeros. Pools have any
    strides, 1 for the last dimension, and no two elements in one place.

    rope: float32 [positions, rot], the cosines of a position's rot / 2 angles, then their sines; the
    first rot elements of each head are rotated, in pairs x[j], x[j + rot / 2], or, interleaved, x[2 j],
    x[2 j + 1]. A position outside rope comes out as NaN. All of one type (float32, float16, bfloat16)."""
    fn = "paged_kv_append"
    # (checks are compared in bulk; what differs is looked at by the helpers, which convert or refuse. A call's
    # host time is most of what appending a decode step takes: 15.4 us a call with the helpers alone)
    ks, ps, dt, int32_t = k.shape, k_pool.shape, k.dtype, torch.int32
    if len(ks) != 3 or v.shape != ks:
        raise ValueError(f"{fn}: k {tuple(ks)}, v {tuple(v.shape)}: expected two [tokens, kv_heads, head_dim]")
    T, Hkv, D = ks
    kv_sb, kv_sh, kv_st = pools(k_pool, v_pool, fn, write=True)
    num_blocks, Hp, block_size, Dp = ps
    if Hp != Hkv or Dp != D:
        raise ValueError(f"{fn}: k {tuple(ks)}, pools {tuple(ps)}: heads or head dims differ")
    if k_pool.dtype != dt or v.dtype != dt or q is not None and q.dtype != dt:
        raise TypeError(f"{fn}: q, k, v and the pools must have one dtype, got {q.dtype if q is not None else None}, {dt}, "
                        f"{v.dtype}, {k_pool.dtype}")
    Hq = 0
    if q is not None:
        qs = q.shape
        if len(qs) != 3 or qs[0] != T or qs[2] != D:
            raise ValueError(f"{fn}: q {tuple(qs)} for k {tuple(ks)}")
        Hq = qs[1]
    rot = positions = rope_ld = 0
    if rope is not None:
        if rope.dim() != 2 or rope.dtype != torch.float32:
            raise ValueError(f"{fn}: rope must be float32 [positions, rot], got {rope.dtype} {tuple(rope.shape)}")
        positions, rot = rope.shape
        if rot % 2 or rot > D:
            raise ValueError(f"{fn}: rope rotates {rot} of {D} elements: an even number up to the head dim is needed")
        if not positions and rot:
            rope = rope.new_empty(1, rot)  # (an address: that of no elements is null. No row of it counts)
        rope_ld, inner = rope.stride()
        if inner != 1 or rope_ld < rot:
            rope = rope.contiguous()
            rope_ld = rot
    n = context_lens.shape[0] if context_lens.dim() == 1 else -1
    if context_lens.dtype != int32_t or n < 0 or context_lens.stride(0) != 1:
        context_lens = int32(context_lens, "context_lens", fn, (None,))
    ts = block_tables.shape
    if block_tables.dtype != int32_t or len(ts) != 2 or ts[0] != n or block_tables.stride(1) != 1:
        block_tables = int32(block_tables, "block_tables", fn, (n, None))
    if cu_seqlens is not None:
        if cu_seqlens.dtype != int32_t or cu_seqlens.shape != (n + 1,) or cu_seqlens.stride(0) != 1:
            cu_seqlens = int32(cu_seqlens, "cu_seqlens", fn, (n + 1,))
    elif n != T:
        raise ValueError(f"{fn}: {T} rows for {n} sequences: without cu_seqlens, each has one")
    if torch.is_grad_enabled() or forward_ad._current_level >= 0:
        no_grad_of(fn, q, k, v, k_pool, v_pool, rope)
    dev = one_device(fn, k, v, k_pool, v_pool, block_tables, context_lens, q, cu_seqlens, rope)
    k_st, k_sh, inner = k.stride()
    if inner != 1 and D > 1:
        k = k.contiguous()
        k_st, k_sh, _ = k.stride()
    v_st, v_sh, inner = v.stride()
    if inner != 1 and D > 1:
        v = v.contiguous()
        v_st, v_sh, _ = v.stride()
    turn = q is not None and rot > 0
    out, q_st, q_sh, q_at, out_at = q, 0, 0, 0, 0
    if turn:
        q_st, q_sh, inner = q.stride()
        if inner != 1 and D > 1:
            q = q.contiguous()
            q_st, q_sh, _ = q.stride()
        out = fresh(q, (T, Hq, D))
        q_at, out_at = q.data_ptr(), out.data_ptr()
    rc = kernels.lib().mlsx_paged_append(_ARGS.pack(
        q_at, k.data_ptr(), v.data_ptr(), k_pool.data_ptr(), v_pool.data_ptr(), out_at, block_tables.data_ptr(),
        context_lens.data_ptr(), 0 if cu_seqlens is None else cu_seqlens.data_ptr(), rope.data_ptr() if rot else 0,
        _DT[dt] if dt in _DT else dt_code(dt, fn), q_st, q_sh, k_st, k_sh, v_st, v_sh, kv_sb, kv_sh, kv_st,
        block_tables.stride(0), rope_ld, num_blocks, n, T, Hq, Hkv, D, block_size, block_tables.shape[1], positions if rot else 0, rot,
        interleaved), _raw_stream(dev))
    if rc:
        kernels.check(rc, fn)
    return out
