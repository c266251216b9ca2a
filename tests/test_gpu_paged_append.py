"""paged_kv_append against its 64-bit form. Tolerance: a rotated value is two products and a sum in fp32 (3 roundings
of 2^-24 of |a| + |b|) and one rounding to its type (eps / 2 of the value); copies are exact."""

from __future__ import annotations

import pytest
import torch

from paged_plain import offsets

from kernels.paged_kv import paged_kv_append

pytestmark = pytest.mark.gpu

BF, HF, FP = torch.bfloat16, torch.float16, torch.float32


def _rope(P, rot):
    ang = torch.arange(P, dtype=torch.float64)[:, None] * 10000.0 ** (-2.0 * torch.arange(rot // 2, dtype=torch.float64) / max(rot, 1))
    return torch.cat([ang.cos(), ang.sin()], 1).float().cuda()


def _turn(x, rope, pos, inter):
    """(rotated [.., D] in 64 bits, the sum of the products' sizes); pos inside rope."""
    rot = rope.shape[1]
    c, s = (t[:, None].double() for t in (rope[pos, :rot // 2], rope[pos, rot // 2:]))
    x = x.double()
    r = x[..., :rot]
    a, b = (r[..., 0::2], r[..., 1::2]) if inter else (r[..., :rot // 2], r[..., rot // 2:])
    y, z = a * c - b * s, a * s + b * c
    m, w = (a * c).abs() + (b * s).abs(), (a * s).abs() + (b * c).abs()
    join = (lambda p, q: torch.stack([p, q], -1).flatten(-2)) if inter else (lambda p, q: torch.cat([p, q], -1))
    rest = x[..., rot:]
    return torch.cat([join(y, z), rest], -1), torch.cat([join(m, w), torch.zeros_like(rest)], -1)


def _case(new, past, Hq, Hkv, D, bs, dtype, seed=0):
    g = torch.Generator().manual_seed(seed)
    lens = [a + b for a, b in zip(new, past)]
    need = [-(-n // bs) for n in lens]
    ids = torch.randperm(sum(need) + 2, generator=g).to(torch.int32)
    tab, at = torch.full((len(new), max(need) + 1), -1, dtype=torch.int32), 0
    for i, u in enumerate(need):
        tab[i, :u] = ids[at:at + u]
        at += u
    T = sum(new)
    q, k, v = (torch.randn(T, h, D, generator=g).to(dtype).cuda() for h in (Hq, Hkv, Hkv))
    kp, vp = (torch.randn(sum(need) + 2, Hkv, bs, D, generator=g).to(dtype).cuda() for _ in range(2))
    return q, k, v, kp, vp, tab.cuda(), torch.tensor(lens, dtype=torch.int32).cuda()


def _near(y, want, size):
    u = torch.finfo(y.dtype).eps / 2
    tiny = torch.finfo(y.dtype).smallest_normal * u  # half the smallest step
    over = (y.double() - want).abs() - (u * want.abs() * 1.01 + 3 * 2.0 ** -24 * size + tiny)
    assert float(over.max()) <= 0, float(over.max())


@pytest.mark.parametrize("dtype", [BF, HF, FP])
@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("Hq,Hkv,D,rot,bs,new,past", [
    (32, 8, 128, 128, 16, [1] * 9, [0, 1, 15, 16, 17, 100, 4000, 31, 2]),
    (4, 2, 128, 64, 16, [1, 40, 0, 300, 7], [0, 0, 9, 33, 100]),
    (7, 1, 80, 80, 24, [5, 17], [3, 0]), (3, 3, 80, 40, 8, [2, 2, 2], [7, 8, 0]), (2, 1, 256, 128, 1, [3, 1], [0, 5]),
    (2, 2, 33, 6, 5, [4, 9], [1, 0]), (1, 1, 2, 2, 3, [2], [0]), (5, 2, 20, 10, 16, [6], [11]),
    (2, 1, 1024, 1024, 16, [3], [2]), (1, 1, 600, 300, 16, [2], [0]),
])
def test_against_the_formula(dev, dtype, inter, Hq, Hkv, D, rot, bs, new, past):
    q, k, v, kp, vp, tab, ctx = _case(new, past, Hq, Hkv, D, bs, dtype)
    rope = _rope(int(ctx.max()), rot)
    k0, v0 = kp.clone(), vp.clone()
    cu = None if set(new) == {1} else offsets(new)
    out = paged_kv_append(q, k, v, kp, vp, tab, ctx, cu, rope=rope, interleaved=inter)
    pos = torch.cat([torch.arange(p, p + n) for n, p in zip(new, past)]).cuda()
    seq = torch.repeat_interleave(torch.arange(len(new)), torch.tensor(new)).cuda()
    _near(out, *_turn(q, rope, pos, inter))
    blk, off = tab[seq, pos // bs].long(), pos % bs
    _near(kp[blk, :, off], *_turn(k, rope, pos, inter))
    assert torch.equal(vp[blk, :, off], v)
    k0[blk, :, off], v0[blk, :, off] = kp[blk, :, off], vp[blk, :, off]
    assert torch.equal(kp, k0) and torch.equal(vp, v0)  # nothing else is written


@pytest.mark.parametrize("dtype,D", [(BF, 64), (FP, 33)])
def test_without_rotation_and_without_queries(dev, dtype, D):
    new, past = [3, 1, 20], [0, 5, 30]
    q, k, v, kp, vp, tab, ctx = _case(new, past, 4, 2, D, 16, dtype)
    pos = torch.cat([torch.arange(p, p + n) for n, p in zip(new, past)]).cuda()
    seq = torch.repeat_interleave(torch.arange(3), torch.tensor(new)).cuda()
    blk, off = tab[seq, pos // 16].long(), pos % 16
    assert paged_kv_append(q, k, v, kp, vp, tab, ctx, offsets(new)) is q
    assert torch.equal(kp[blk, :, off], k) and torch.equal(vp[blk, :, off], v)
    kp.zero_()
    rope = _rope(64, D // 2 * 2)
    assert paged_kv_append(None, k, v, kp, vp, tab, ctx, offsets(new), rope=rope) is None
    _near(kp[blk, :, off], *_turn(k, rope, pos, False))
    assert paged_kv_append(q, k, v, kp, vp, tab, ctx, offsets(new), rope=rope[:, :0]) is q


def test_rows_without_a_place(dev):
    """Bad block ids, positions outside the table, lengths below the rows, rows of no sequence."""
    new, past = [4, 40, 3], [0, 0, 0]
    q, k, v, kp, vp, tab, ctx = _case(new, past, 2, 1, 64, 16, BF)
    lead, T = 2, 2 + 47 + 6
    q, k, v = (torch.randn(T, h, 64, device=dev).to(BF) for h in (2, 1, 1))
    tab[1, 1], tab[0, 0] = kp.shape[0], -1
    ctx = torch.tensor([4, 40, 1], dtype=torch.int32, device=dev)  # the third: rows at -2, -1 and 0
    rope = _rope(30, 64)                                           # the second: positions 30 on are outside
    k0, v0 = kp.clone(), vp.clone()
    out = paged_kv_append(q, k, v, kp, vp, tab[:, :2].contiguous(), ctx, offsets(new, lead=lead), rope=rope)
    assert bool((out[:lead] == 0).all()) and bool((out[lead + 47:] == 0).all())
    assert bool(torch.isnan(out[lead + 4 + 30:lead + 4 + 42]).all()) and bool(torch.isfinite(out[lead:lead + 34]).all())
    assert bool(torch.isfinite(out[lead + 46]).all())
    b1, b2 = int(tab[1, 0]), int(tab[2, 0])
    assert torch.equal(vp[b1, 0], v[lead + 4:lead + 20, 0]) and torch.equal(vp[b2, 0, 0], v[lead + 46, 0])
    k0[b1], v0[b1], k0[b2, 0, 0], v0[b2, 0, 0] = kp[b1], vp[b1], kp[b2, 0, 0], vp[b2, 0, 0]
    assert torch.equal(kp, k0) and torch.equal(vp, v0)


@pytest.mark.parametrize("dtype", [BF, FP])
def test_strides_streams_and_graphs(dev, dtype):
    """Slices of one fused projection, token-major pools, 64-bit indexes; on a side stream, and replayed."""
    new, past = [9, 1, 30], [20, 7, 0]
    q, k, v, kp, vp, tab, ctx = _case(new, past, 6, 2, 64, 16, dtype)
    rope, cu = _rope(64, 64), offsets(new)
    a, b = kp.clone(), vp.clone()
    want = paged_kv_append(q, k, v, a, b, tab, ctx, cu, rope=rope)
    fused = torch.cat([q, k, v], 1)
    tm = [t.transpose(1, 2).contiguous().transpose(1, 2) for t in (kp, vp)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = paged_kv_append(fused[:, :6], fused[:, 6:8], fused[:, 8:], *tm, tab.long(), ctx.long(), cu.long(), rope=rope)
    side.synchronize()
    assert torch.equal(got, want) and torch.equal(tm[0], a) and torch.equal(tm[1], b)
    odd = torch.zeros(40, 10, 67, dtype=dtype, device=dev)
    odd[..., 1:65] = fused
    c, d = kp.clone(), vp.clone()
    got = paged_kv_append(odd[:, :6, 1:65], odd[:, 6:8, 1:65], odd[:, 8:, 1:65], c, d, tab, ctx, cu, rope=rope)
    assert torch.equal(got, want) and torch.equal(c, a) and torch.equal(d, b)
    c, d = kp.clone(), vp.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = paged_kv_append(q, k, v, c, d, tab, ctx, cu, rope=rope)
    for _ in range(3):
        c.copy_(kp), d.copy_(vp), got.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, want) and torch.equal(c, a) and torch.equal(d, b)


def test_past_32_bits(dev):
    blocks = 1 << 18
    kp = torch.empty(blocks, 2, 64, 128, dtype=BF, device=dev)  # 8 GiB
    vp = torch.empty_like(kp)
    tab = torch.tensor([[blocks - 1], [blocks // 2 + 3]], dtype=torch.int32, device=dev)
    k, v = (torch.randn(2, 2, 128, device=dev).to(BF) for _ in range(2))
    paged_kv_append(None, k, v, kp, vp, tab, torch.tensor([64, 1], dtype=torch.int32, device=dev))
    assert torch.equal(kp[blocks - 1, :, 63], k[0]) and torch.equal(vp[blocks // 2 + 3, :, 0], v[1])


def test_many_sequences(dev):
    new = [1 + i % 4 for i in range(900)]
    q, k, v, kp, vp, tab, ctx = _case(new, [i % 50 for i in range(900)], 2, 1, 64, 16, BF)
    pos = torch.cat([torch.arange(p, p + n) for n, p in zip(new, [i % 50 for i in range(900)])]).cuda()
    seq = torch.repeat_interleave(torch.arange(900), torch.tensor(new)).cuda()
    paged_kv_append(None, k, v, kp, vp, tab, ctx, offsets(new))
    assert torch.equal(vp[tab[seq, pos // 16].long(), :, pos % 16], v)


def test_nothing_to_append(dev):
    q, k, v, kp, vp, tab, ctx = _case([1, 1], [0, 0], 2, 1, 64, 16, BF)
    k0 = kp.clone()
    out = paged_kv_append(q[:0], k[:0], v[:0], kp, vp, tab, ctx, offsets([0, 0]), rope=_rope(4, 64))
    assert out.shape == (0, 2, 64) and torch.equal(kp, k0)
