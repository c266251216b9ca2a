"""paged_attention and shared_prefix_attention against their 64-bit forms: types, head layouts, lengths from one
token on, block sizes, strides, masks that leave rows empty, and values in places that no row sees.
Tolerances: paged_plain.attention's bound."""

from __future__ import annotations

import pytest
import torch

from paged_plain import attention, cache, check, offsets

from kernels.paged_attention import paged_attention, paged_attention_decode, shared_prefix_attention

pytestmark = pytest.mark.gpu

BF, HF, FP = torch.bfloat16, torch.float16, torch.float32


def _q(T, H, D, dtype, seed=5):
    return torch.randn(T, H, D, generator=torch.Generator().manual_seed(seed)).to(dtype).cuda()


def _slopes(H):
    return torch.tensor([2.0 ** (-8 * (h + 1) / H) for h in range(H)], dtype=torch.float32).cuda()


@pytest.mark.parametrize("dtype", [BF, HF, FP])
@pytest.mark.parametrize("D,kvh,group,bs", [(128, 2, 4, 16), (64, 1, 1, 8), (80, 2, 7, 24), (256, 1, 2, 16), (96, 3, 8, 1),
                                            (8, 2, 3, 5), (200, 1, 16, 64), (40, 1, 20, 32), (33, 2, 2, 16), (1, 1, 5, 7)])
def test_single_tokens(dev, dtype, D, kvh, group, bs):
    lens = [1, 2, bs, bs + 1, 0, 129, 700]
    kp, vp, tab, ctx = cache(lens, kvh, D, bs, dtype, D)
    q = _q(len(lens), kvh * group, D, dtype)
    check(paged_attention(q, kp, vp, tab, ctx), *attention(q, kp, vp, tab, lens), f"{dtype} D={D}")


@pytest.mark.parametrize("dtype", [BF, HF, FP])
@pytest.mark.parametrize("D,kvh,group,bs", [(128, 2, 4, 16), (64, 8, 1, 16), (80, 1, 7, 24), (256, 2, 2, 16), (96, 1, 8, 1),
                                            (24, 2, 3, 5), (50, 1, 2, 32)])
@pytest.mark.parametrize("opts", ["plain", "cap", "slopes_window", "prefix", "all"])
def test_prompts_and_chunks(dev, dtype, D, kvh, group, bs, opts):
    new, past = [1, 65, 0, 130, 17, 3], [0, 100, 50, 0, 333, 5]
    lens = [a + b for a, b in zip(new, past)]
    kp, vp, tab, ctx = cache(lens, kvh, D, bs, dtype, 1)
    q = _q(sum(new), kvh * group, D, dtype)
    o = {}
    if opts in ("cap", "all"):
        o["softcap"] = 5.0
    if opts in ("slopes_window", "all"):
        o["slopes"], o["window"] = _slopes(kvh * group), 40
    if opts in ("prefix", "all"):
        o["prefix_lens"] = torch.tensor([1, 20, 7, 90, 400, 0], dtype=torch.int32, device=dev)
    want = attention(q, kp, vp, tab, lens, new, **o)
    for hint in (None, 4, max(new)):  # a hint that is wrong chooses another kernel, not another result
        check(paged_attention(q, kp, vp, tab, ctx, offsets(new), max_new=hint, **o), *want, f"{opts} {hint}")


@pytest.mark.parametrize("dtype,D", [(BF, 128), (FP, 64), (HF, 256)])
@pytest.mark.parametrize("kvh,group", [(8, 1), (1, 8), (2, 12)])
@pytest.mark.parametrize("lens,new", [([5000], [1]), ([4100, 3, 800], [9, 2, 5]), ([40] * 70 + [3000], None),
                                      ([2300], [300]), ([900] * 3, [200, 1, 30])])
def test_long_contexts_in_pieces(dev, dtype, D, kvh, group, lens, new):
    kp, vp, tab, ctx = cache(lens, kvh, D, 16, dtype, 2, wide=9)
    T = sum(new) if new else len(lens)
    q = _q(T, kvh * group, D, dtype)
    cu = offsets(new) if new and max(new) > 1 else None
    y = paged_attention(q, kp, vp, tab, ctx, cu)
    check(y, *attention(q, kp, vp, tab, lens, new), "pieces")
    assert torch.equal(y, paged_attention(q, kp, vp, tab, ctx, cu))  # no order of joining changes


def test_many_sequences(dev):
    """Past the sequences whose lengths the kernels sum, and past one round of the search."""
    lens = [1 + (37 * i) % 90 for i in range(1500)]
    kp, vp, tab, ctx = cache(lens, 1, 64, 16, BF, 3)
    q = _q(len(lens), 4, 64, BF)
    check(paged_attention(q, kp, vp, tab, ctx), *attention(q, kp, vp, tab, lens), "decode")
    new = [min(n, 1 + i % 3) for i, n in enumerate(lens)]
    q = _q(sum(new), 4, 64, BF)
    check(paged_attention(q, kp, vp, tab, ctx, offsets(new)), *attention(q, kp, vp, tab, lens, new), "ragged")


@pytest.mark.parametrize("dtype,D", [(BF, 128), (FP, 64), (HF, 80)])
@pytest.mark.parametrize("new", [[1, 1, 1, 1], [3, 40, 9, 200]])
def test_rows_that_see_nothing(dev, dtype, D, new):
    """Fewer cached tokens than rows, none at all, a negative length, and rows of no sequence."""
    lens = [0, 25, -3, 100]
    kp, vp, tab, ctx = cache(lens, 2, D, 16, dtype, 4)
    T = 5 + sum(new) + 70
    q = _q(T, 4, D, dtype)
    want, bound = attention(q, kp, vp, tab, lens, new, lead=5)
    y = paged_attention(q, kp, vp, tab, ctx, offsets(new, lead=5))
    check(y, want, bound)
    assert bool((y[:5] == 0).all()) and bool((y[5 + sum(new):] == 0).all())
    pl = torch.tensor([9, 30, 4, -2], dtype=torch.int32, device=dev)
    check(paged_attention(q, kp, vp, tab, ctx, offsets(new, lead=5), prefix_lens=pl, window=3),
          *attention(q, kp, vp, tab, lens, new, lead=5, prefix_lens=pl, window=3))


@pytest.mark.parametrize("new", [[1, 1, 1], [20, 90, 2]])
def test_tables_with_holes_and_ends(dev, new):
    """Block ids outside the pool hold no tokens; a context past its table is cut there, the positions are not."""
    lens = [400, 300, 90]
    kp, vp, tab, ctx = cache(lens, 2, 128, 16, BF, 6)
    tab[0, 3], tab[0, 24], tab[1, 0], tab[2, :] = -1, kp.shape[0], 2 ** 31 - 1, -2 ** 31
    q = _q(sum(new), 8, 128, BF)
    cu = offsets(new) if max(new) > 1 else None
    for w in (0, 150):
        check(paged_attention(q, kp, vp, tab, ctx, cu, window=w), *attention(q, kp, vp, tab, lens, new, window=w))
        short = tab[:, :15]
        check(paged_attention(q, kp, vp, short, ctx, cu, window=w), *attention(q, kp, vp, short, lens, new, window=w))
    empty = tab[:, :0]
    assert bool((paged_attention(q, kp, vp, empty, ctx, cu) == 0).all())


@pytest.mark.parametrize("dtype,D", [(BF, 128), (FP, 64), (HF, 72), (FP, 256)])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_values_in_slots_that_hold_no_token(dev, dtype, D, bad):
    """Past a context's end, before a window, and in unused blocks."""
    lens, new = [37, 100, 1, 260], [1, 1, 1, 1]
    kp, vp, tab, ctx = cache(lens, 2, D, 16, dtype, 7)
    clean = kp.clone(), vp.clone()
    used = torch.zeros(kp.shape[0], 16, dtype=torch.bool)
    for i, n in enumerate(lens):
        for t in range(max(0, n - 30), n):
            used[int(tab[i, t // 16]), t % 16] = True
    used = used.to(dev)[:, None, :, None]
    kp, vp = (torch.where(used, t, torch.full_like(t, bad)) for t in clean)
    q = _q(4, 4, D, dtype)
    check(paged_attention(q, kp, vp, tab, ctx, window=30), *attention(q, *clean, tab, lens, window=30))


@pytest.mark.parametrize("dtype,D", [(BF, 128), (FP, 64), (BF, 256)])
@pytest.mark.parametrize("n,kvh,group,shared", [(1, 2, 4, 100), (4, 8, 4, 1000), (30, 2, 8, 513), (200, 1, 4, 2100), (3, 2, 1, 0)])
@pytest.mark.parametrize("opts", ["plain", "all"])
def test_shared_prefix(dev, dtype, D, n, kvh, group, shared, opts):
    bs = 16
    lens = [(17 * i) % 60 for i in range(n)]  # (0: no token of its own)
    kp, vp, tab, ctx = cache(lens + [shared], kvh, D, bs, dtype, 8)
    pre, tab, ctx = tab[n, :-(-shared // bs)].contiguous(), tab[:n], ctx[:n]
    q = _q(n, kvh * group, D, dtype)
    o = dict(softcap=20.0, slopes=_slopes(kvh * group), window=shared // 2 + 3) if opts == "all" else {}
    y = shared_prefix_attention(q, kp, vp, pre, shared, tab, ctx, **o)
    check(y, *attention(q, kp, vp, tab, lens, shared=pre, shared_len=shared, **o), opts)


def test_shared_prefix_with_holes(dev):
    lens, shared = [5, 0, 33], 200
    kp, vp, tab, ctx = cache(lens + [shared], 2, 64, 16, BF, 9)
    pre, tab, ctx = tab[3].clone(), tab[:3], ctx[:3]
    pre[2], pre[7] = -1, kp.shape[0]
    q = _q(3, 4, 64, BF)
    check(shared_prefix_attention(q, kp, vp, pre, shared, tab, ctx),
          *attention(q, kp, vp, tab, lens, shared=pre, shared_len=shared))


@pytest.mark.parametrize("dtype", [BF, FP])
def test_strides_and_orders(dev, dtype):
    """Pools kept token-major, heads of q inside a fused projection, tables as columns of a wider one, slices at odd
    addresses (element loads), index tensors of 64 bits."""
    lens, new = [70, 200, 3], [33, 1, 3]
    kp, vp, tab, ctx = cache(lens, 2, 64, 16, dtype, 10)
    q = _q(sum(new), 6, 64, dtype)
    cu = offsets(new)
    want = attention(q, kp, vp, tab, lens, new)
    tm = [t.transpose(1, 2).contiguous().transpose(1, 2) for t in (kp, vp)]
    fused = torch.zeros(sum(new), 10, 64, dtype=dtype, device=dev)
    fused[:, 2:8] = q
    wide = torch.full((3, tab.shape[1] + 4), -1, dtype=torch.int32, device=dev)
    wide[:, 2:-2] = tab
    check(paged_attention(fused[:, 2:8], *tm, wide[:, 2:-2], ctx, cu), *want)
    odd = [torch.zeros(*t.shape[:3], 67, dtype=dtype, device=dev) for t in (kp, vp)]
    for a, b in zip(odd, (kp, vp)):
        a[..., 1:65] = b
    oq = torch.zeros(sum(new), 6, 65, dtype=dtype, device=dev)
    oq[..., 1:] = q
    check(paged_attention(oq[..., 1:], odd[0][..., 1:65], odd[1][..., 1:65], tab.long(), ctx.long(), cu.long()), *want)
    dq = q.transpose(1, 2).contiguous().transpose(1, 2)  # inner stride not 1
    check(paged_attention(dq, kp, vp, tab.T.contiguous().T, ctx, cu), *want)


def test_offsets_past_32_bits(dev):
    """Blocks beyond 4 GiB of a pool."""
    blocks, bs, D = 1 << 18, 64, 128
    kp = torch.empty(blocks, 2, bs, D, dtype=BF, device=dev)  # 8 GiB
    vp = torch.empty_like(kp)
    ids = [blocks - 1, 5, blocks // 2 + 1, blocks - 7]
    small = torch.tensor(ids)
    g = torch.Generator().manual_seed(0)
    ks, vs = (torch.randn(4, 2, bs, D, generator=g).to(BF).to(dev) for _ in range(2))
    kp[small.to(dev)], vp[small.to(dev)] = ks, vs
    tab = torch.tensor([ids], dtype=torch.int32, device=dev)
    tab4 = torch.arange(4, dtype=torch.int32, device=dev)[None]
    for new in (1, 70):
        q = _q(new, 8, D, BF)
        want = attention(q, ks, vs, tab4, [250], [new])
        cu = offsets([new])
        check(paged_attention(q, kp, vp, tab, torch.tensor([250], dtype=torch.int32, device=dev), cu), *want)


def test_one_head_a_kv_head_agrees_with_the_decode_kernel(dev):
    lens = [300, 1, 77]
    kp, vp, tab, ctx = cache(lens, 4, 64, 16, FP, 11)
    q = _q(3, 4, 64, FP)
    a, b = paged_attention(q, kp, vp, tab, ctx), paged_attention_decode(q, kp, vp, tab, ctx)
    _, bound = attention(q, kp, vp, tab, lens)
    assert bool(((a.double() - b.double()).abs() <= 2 * bound).all())


@pytest.mark.parametrize("scale", [-0.3, 0.0, 2.0])
def test_scales(dev, scale):
    lens, new = [100, 9], [40, 9]
    kp, vp, tab, ctx = cache(lens, 2, 64, 16, FP, 12)
    q = _q(sum(new), 4, 64, FP)
    check(paged_attention(q, kp, vp, tab, ctx, offsets(new), scale=scale), *attention(q, kp, vp, tab, lens, new, scale=scale))


def test_scores_of_any_size(dev):
    """Scores near 3e4, where only one key weighs, and a reference that rises from tile to tile."""
    lens = [500]
    kp, vp, tab, ctx = cache(lens, 1, 64, 16, FP, 13)
    for t in range(500):
        kp[int(tab[0, t // 16]), 0, t % 16] *= t
    q = _q(1, 4, 64, FP)
    y = paged_attention(q, kp, vp, tab, ctx, scale=4.0)
    want, bound = attention(q, kp, vp, tab, lens, scale=4.0)
    check(y, want, bound)
    assert bool(torch.isfinite(y).all())


def test_on_another_stream_and_in_a_graph(dev):
    lens, new = [600, 90, 41], [5, 1, 40]
    kp, vp, tab, ctx = cache(lens, 2, 128, 16, BF, 14)
    q = _q(sum(new), 8, 128, BF)
    cu = offsets(new)
    pre = tab[0, :20].contiguous()
    q3 = _q(3, 8, 128, BF)
    eager = paged_attention(q, kp, vp, tab, ctx, cu), shared_prefix_attention(q3, kp, vp, pre, 300, tab, ctx)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = paged_attention(q, kp, vp, tab, ctx, cu), shared_prefix_attention(q3, kp, vp, pre, 300, tab, ctx)
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = paged_attention(q, kp, vp, tab, ctx, cu), shared_prefix_attention(q3, kp, vp, pre, 300, tab, ctx)
    for a, b in zip(eager, other):
        assert torch.equal(a, b)
    for _ in range(3):
        for t in got:
            t.zero_()
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(eager, got):
            assert torch.equal(a, b)
        paged_attention(q, kp, vp, tab, ctx, cu)  # eager work between replays
    ctx.copy_(torch.tensor([333, 80, 41], dtype=torch.int32))  # other lengths, the same graph
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(got[0], paged_attention(q, kp, vp, tab, ctx, cu))


def test_empty_calls(dev):
    kp, vp, tab, ctx = cache([4, 9], 2, 64, 16, BF, 15)
    q = _q(0, 4, 64, BF)
    assert paged_attention(q, kp, vp, tab, ctx, offsets([0, 0])).shape == (0, 4, 64)
    assert paged_attention(q, kp, vp, tab[:0], ctx[:0]).shape == (0, 4, 64)
    assert bool((paged_attention(_q(3, 4, 64, BF), kp, vp, tab[:0], ctx[:0], offsets([])) == 0).all())


@pytest.mark.parametrize("dtype,D,group", [(BF, 128, 4), (HF, 64, 1), (FP, 64, 2), (BF, 256, 2), (FP, 128, 1), (HF, 80, 3)])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("new,past", [([200, 9], [0, 40]), ([5, 3], [60, 0]), ([40], [300]), ([300], [70])])
def test_values_that_only_later_rows_see(dev, dtype, D, group, bad, new, past):
    """A cached value that is no number reaches the rows that see its token, in its own element, and no others."""
    lens = [a + b for a, b in zip(new, past)]
    for window in (0, 25):
        kp, vp, tab, ctx = cache(lens, 1, D, 16, dtype, 21)
        q = _q(sum(new), group, D, dtype)
        want, bound = attention(q, kp, vp, tab, lens, new, window=window)
        row = 0
        for s, (cnt, n) in enumerate(zip(new, lens)):
            for j in (n - 1, n - cnt // 2 - 1, max(0, n - cnt - 3)):
                vp[int(tab[s, j // 16]), 0, j % 16, j % D] = bad
                pos = torch.arange(n - cnt, n, device=dev)
                sees = (pos >= j) & ((pos - j < window) if window else True)
                part = want[row:row + cnt, :, j % D]
                add = torch.full_like(part, bad)
                want[row:row + cnt, :, j % D] = torch.where(sees[:, None], part + add, part)
            row += cnt
        y = paged_attention(q, kp, vp, tab, ctx, offsets(new), window=window).double()
        odd = ~torch.isfinite(want)
        assert bool((~torch.isfinite(y) == odd).all()), f"{int((~torch.isfinite(y) != odd).sum())} elements"
        if bad == bad:
            assert bool((y[odd] == want[odd]).all())
        check(torch.where(odd, 0.0, y), torch.where(odd, 0.0, want), bound.nan_to_num(0.0, 0.0, 0.0) + torch.where(odd, 1e-30, 0.0))
