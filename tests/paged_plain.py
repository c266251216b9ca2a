"""Plain 64-bit forms of the paged serving operators, with the bound that a kernel's rounding may reach."""

from __future__ import annotations

import torch


def cache(lens, kv_heads, D, bs, dtype, seed, extra=3, wide=0, device="cuda"):
    """Pools with each sequence's tokens in shuffled blocks; unused table entries are invalid ids."""
    g = torch.Generator().manual_seed(seed)
    need = [-(-max(n, 0) // bs) for n in lens]
    ids = torch.randperm(sum(need) + extra, generator=g).to(torch.int32)
    tab, at = torch.full((len(lens), max(need, default=0) + wide), -7, dtype=torch.int32), 0
    for i, u in enumerate(need):
        tab[i, :u] = ids[at:at + u]
        at += u
    shape = (sum(need) + extra, kv_heads, bs, D)
    k, v = (torch.randn(*shape, generator=g).to(dtype).to(device) for _ in range(2))
    return k, v, tab.to(device), torch.tensor(lens, dtype=torch.int32, device=device)


def offsets(new, lead=0, device="cuda"):
    cu = [lead]
    for x in new:
        cu.append(cu[-1] + x)
    return torch.tensor(cu, dtype=torch.int32, device=device)


def gather(pool, ids, n):
    """[kv_heads, n, D] in 64 bits, and which of the tokens have a block; the others are zeros."""
    ids = ids.long()
    ok = (ids >= 0) & (ids < pool.shape[0])
    x = pool[ids.clamp(0, pool.shape[0] - 1)].double()
    x = x.transpose(0, 1).reshape(pool.shape[1], -1, pool.shape[3])[:, :n]
    there = ok.repeat_interleave(pool.shape[2])[:n]
    return torch.where(there[None, :, None], x, 0.0), there


def attention(q, kp, vp, tab, lens, new=None, lead=0, *, scale=None, softcap=0.0, slopes=None, window=0, prefix_lens=None,
              shared=None, shared_len=0):
    """(result, bound) of paged_attention, or with `shared` of shared_prefix_attention. new: rows of each
    sequence (None: one each), from row `lead` on.

    The bound: the result's own rounding (half a step of its type, eps / 2 of the value), each weight's
    rounding to a 16-bit type (eps / 2 of the weights' share of |v|), and what fp32 loses in a score, which
    changes its weight by as much: products of D terms and the cap (tanh to 2^-22) or bias, 2^-24 of the largest a
    step; sums over the keys. fp16 weights under 2^-24 of the largest 2^8 lose half their last step."""
    T, H, D = q.shape
    bs, kvh = kp.shape[2], kp.shape[1]
    u = torch.finfo(q.dtype).eps / 2
    scale = D ** -0.5 if scale is None else scale
    new = [1] * len(lens) if new is None else new
    out = torch.zeros(T, H, D, dtype=torch.float64, device=q.device)
    bound = torch.full_like(out, 1e-35)
    row = lead
    for s, cnt in enumerate(new):
        n = int(lens[s])
        have = min(max(n, 0), tab.shape[1] * bs)
        k, there = gather(kp, tab[s, :-(-have // bs)], have)
        v, _ = gather(vp, tab[s, :-(-have // bs)], have)
        pos = torch.arange(n - cnt, n, device=q.device)
        if shared is not None:
            k0, t0 = gather(kp, shared[:-(-shared_len // bs)], shared_len)
            k, there = torch.cat([k0, k], 1), torch.cat([t0, there])
            v = torch.cat([gather(vp, shared[:-(-shared_len // bs)], shared_len)[0], v], 1)
            pos = pos.clamp(min=-1) + shared_len
        j = torch.arange(k.shape[1], device=q.device)
        gap = pos[:, None] - j
        see = gap >= 0
        if prefix_lens is not None:
            see = see | (j < int(prefix_lens[s]))
        if window:
            see = see & (gap < window)
        see = see & there
        if cnt and k.shape[1]:
            for h in range(H):
                kk, vv, qq = k[h // (H // kvh)], v[h // (H // kvh)], q[row:row + cnt, h].double()
                x = (qq @ kk.T) * scale
                loss = (D + 8) * 2.0 ** -24 * ((qq.abs() @ kk.abs().T) * abs(scale)).max()
                if softcap:
                    x = softcap * torch.tanh(x / softcap)
                    loss = loss + softcap * 2.0 ** -21
                if slopes is not None:
                    x = x - slopes[h].double() * gap.abs()
                loss = loss + 2.0 ** -22 * x.abs().max()
                x = x.masked_fill(~see, float("-inf"))
                p = torch.nan_to_num(torch.softmax(x, -1), nan=0.0)
                p = torch.where(see, p, 0.0)
                vs = torch.where(see.any(0)[:, None], vv, 0.0)
                out[row:row + cnt, h] = p @ vs
                share = (1.02 * u if q.dtype != torch.float32 else 0.0) + 2 * loss + k.shape[1] * 2.0 ** -23
                bound[row:row + cnt, h] += share * (p @ vs.abs()) + k.shape[1] * 2.0 ** -32 * vs.abs().max()
        row += cnt
    return out, bound + u * 1.01 * out.abs()


def check(y, want, bound, what=""):
    assert y.shape == want.shape
    over = (y.double() - want).abs() - bound
    assert bool((over <= 0).all()), f"{what}: {int((~(over <= 0)).sum())} of {over.numel()} off, the worst by " \
                                    f"{float(torch.nan_to_num(over, nan=9e9).max()):.3g} more than {float(bound.max()):.3g}"
