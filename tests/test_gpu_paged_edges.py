"""paged_attention, shared_prefix_attention and paged_kv_append at the edges of what they take: ids outside the
pool deep in a context, views whose heads or tokens share memory, tables and windows at their ends, large caps, and values that are
no numbers. Tolerances: paged_plain.attention's bound where nothing else is said."""

from __future__ import annotations

import pytest
import torch

from paged_plain import attention, cache, check, offsets

import kernels
from kernels._hip import stream
from kernels.paged_attention import _ARGS, paged_attention, shared_prefix_attention
from kernels.paged_kv import paged_kv_append
from serve.paged_layer import PagedAttentionLayer, rope_table

pytestmark = pytest.mark.gpu

BF, HF, FP = torch.bfloat16, torch.float16, torch.float32


def _q(T, H, D, dtype, seed=5):
    return torch.randn(T, H, D, generator=torch.Generator().manual_seed(seed)).to(dtype).cuda()


@pytest.mark.parametrize("dtype,D,bs", [(BF, 128, 16), (HF, 64, 8), (FP, 64, 8), (FP, 256, 16), (BF, 256, 32), (BF, 64, 5), (HF, 33, 16)])
@pytest.mark.parametrize("new", [[1, 1, 1], [3, 4, 2], [50, 20, 33], [200, 70, 150]])
def test_ids_outside_the_pool_deep_in_a_context(dev, dtype, D, bs, new):
    """With more than 1024 sequences a piece is 2048 keys or more: the ids lie 20 to 200 blocks behind its start, before and
    past the registers' first 64, and in a last tile of few keys. (64, 5) and (33, 16) load their tiles by elements."""
    lens = [1500, 21 * bs + 3, 1000] + [0] * 1100
    kp, vp, tab, ctx = cache(lens, 1, D, bs, dtype, 31)
    bad = (-1, -7, kp.shape[0], 2 ** 31 - 1, -2 ** 31)
    for i, at in enumerate((20, 40, 41, 63, 64, 70, 93, 150, 187)):
        if at * bs < lens[0]:
            tab[0, at] = bad[i % 5]
    tab[1, 21] = -1  # the last 3 keys
    tab[2, 1000 // bs - 2], tab[2, 0] = kp.shape[0], -3
    new = new + [0] * 1100 if max(new) > 1 else [1] * len(lens)
    q = _q(sum(new), 4, D, dtype)
    cu = offsets(new) if max(new) > 1 else None
    want = attention(q, kp, vp, tab, lens, new)
    for hint in (None, max(new)):
        check(paged_attention(q, kp, vp, tab, ctx, cu, max_new=hint), *want, f"{hint}")


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("new", [1, 6, 90, 300])
def test_ids_outside_the_pool_in_one_context(dev, dtype, new):
    """The same for a batch of one, in pieces: every id of a run of blocks in turn."""
    lens = [1061]
    kp, vp, tab, ctx = cache(lens, 8, 64, 16, dtype, 32)
    q = _q(new, 16, 64, dtype)
    good = tab.clone()
    for at in (1, 2, 3, 34, 35, 36, 64, 65, 66):
        tab.copy_(good)
        tab[0, at] = -1 - at
        check(paged_attention(q, kp, vp, tab, ctx, offsets([new])), *attention(q, kp, vp, tab, lens, [new]), f"{at}")


@pytest.mark.parametrize("dtype,D", [(BF, 128), (FP, 64), (HF, 50)])
@pytest.mark.parametrize("new", [[1, 1, 1], [30, 200, 2]])
@pytest.mark.parametrize("dim", [0, 1, 2])
def test_expanded_pools(dev, dtype, D, new, dim):
    """One block, head or token seen as several: read as the copy of the view is, and not written."""
    lens = [90, 333, 5]
    kp, vp, tab, ctx = cache(lens, 4, D, 16, dtype, 33)
    kp, vp = (t.narrow(dim, 0, 1).contiguous().expand(t.shape) for t in (kp, vp))  # (the last block's reads end at the storage's end)
    q = _q(sum(new), 8, D, dtype)
    cu = offsets(new) if max(new) > 1 else None
    check(paged_attention(q, kp, vp, tab, ctx, cu), *attention(q, kp, vp, tab, lens, new))
    if cu is None:
        pre = tab[1, :20].contiguous()
        check(shared_prefix_attention(q, kp, vp, pre, 300, tab, ctx), *attention(q, kp, vp, tab, lens, shared=pre, shared_len=300))
    k = _q(sum(new), 4, D, dtype)
    before = kp.clone()
    with pytest.raises(ValueError, match="share memory"):
        paged_kv_append(q, k, k.clone(), kp, vp, tab, ctx, cu)
    assert torch.equal(kp, before)


@pytest.mark.parametrize("dtype,D", [(BF, 128), (FP, 64)])
@pytest.mark.parametrize("cu", [[0, 100, 0, 0], [0, 4000, 0, 0], [50, 10, 90, 20], [4000, 3000, 2000, 0], [-5, 9999, 3, 4001],
                                [3999] * 900 + [0] + [4000] * 900])
@pytest.mark.parametrize("max_new", [1, 40, 4000])
def test_offsets_that_do_not_rise(dev, dtype, D, cu, max_new):
    """Rows are undefined then, but outputs and workspace end where they end, and counts that no tile wrote bound the join."""
    T, H, kvh, guard = 4000, 4, 2, 1 << 16
    n = len(cu) - 1
    kp, vp, tab, ctx = cache([900] * min(n, 3), kvh, D, 16, dtype, 34)
    tab, ctx = (t.repeat(-(-n // 3), *[1] * (t.dim() - 1))[:n].contiguous() for t in (tab, ctx))
    q = _q(T, H, D, dtype)
    off = torch.tensor(cu, dtype=torch.int32, device=dev)
    big = torch.full((T * H * D + 2 * guard,), 3.0, dtype=dtype, device=dev)
    out = big[guard:-guard]
    args = _ARGS.pack(q.data_ptr(), kp.data_ptr(), vp.data_ptr(), tab.data_ptr(), ctx.data_ptr(), off.data_ptr(), 0, 0, 0,
                      out.data_ptr(), {BF: kernels.MLS_BF16, FP: kernels.MLS_F32}[dtype], H * D, D, H * D, D, *kp.stride()[:3],
                      tab.stride(0), kp.shape[0], n, T, kvh, H // kvh, D, 16, tab.shape[1], 0, 0, 0, max_new, D ** -0.5, 0.0)
    need = kernels.lib().mlsx_paged_attention_ws(args)
    work = torch.full((need + 2 * guard,), 0x7F7F7F7F, dtype=torch.int32, device=dev)  # a count far past every record
    kernels.check(kernels.lib().mlsx_paged_attention(args, work[guard:].data_ptr(), need, stream(q.device)), "mlsx_paged_attention")
    torch.cuda.synchronize()
    for t, value in ((big, 3.0), (work, 0x7F7F7F7F)):
        assert bool((t[:guard] == value).all()) and bool((t[-guard:] == value).all())


@pytest.mark.parametrize("dtype,D,cu", [(BF, 128, None), (FP, 64, None), (BF, 128, [0, 300, 500]), (HF, 256, [0, 100, 200])])
def test_a_workspace_that_is_not_needed(dev, dtype, D, cu):
    """A call of one piece writes nothing into a workspace that it is given all the same."""
    lens = [1] * 2000 if cu is None else [300, 200]
    kp, vp, tab, ctx = cache(lens, 2, D, 16, dtype, 37)
    T, n = (len(lens), len(lens)) if cu is None else (cu[-1], 2)
    q, off = _q(T, 8, D, dtype), None if cu is None else torch.tensor(cu, dtype=torch.int32, device=dev)
    out = torch.empty_like(q)
    args = _ARGS.pack(q.data_ptr(), kp.data_ptr(), vp.data_ptr(), tab.data_ptr(), ctx.data_ptr(), 0 if cu is None else off.data_ptr(), 0, 0,
                      0, out.data_ptr(), {BF: kernels.MLS_BF16, HF: kernels.MLS_F16, FP: kernels.MLS_F32}[dtype], 8 * D, D, 8 * D, D,
                      *kp.stride()[:3], tab.stride(0), kp.shape[0], n, T, 2, 4, D, 16, 1 if cu is None else 2, 0, 0, 0, T, D ** -0.5, 0.0)
    assert kernels.lib().mlsx_paged_attention_ws(args) == 0
    work = torch.full((T * 8 * (2 * D + 5),), 7, dtype=torch.int32, device=dev)  # room for what a piece's records would take
    kernels.check(kernels.lib().mlsx_paged_attention(args, work.data_ptr(), work.numel(), stream(q.device)), "mlsx_paged_attention")
    assert bool((work == 7).all())
    new = None if cu is None else [cu[1], cu[2] - cu[1]]
    check(out, *attention(q, kp, vp, tab[:, :1 if cu is None else 2], lens, new))


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("rot", [64, 32])
def test_a_rotation_table_without_rows(dev, dtype, interleaved, rot):
    """Every position is outside it: NaN in the rotated elements of q and k, the others and v as they are."""
    lens = [3, 20]
    kp, vp, tab, ctx = cache(lens, 2, 64, 16, dtype, 35)
    q, k, v = _q(2, 4, 64, dtype, 1), _q(2, 2, 64, dtype, 2), _q(2, 2, 64, dtype, 3)
    table = torch.zeros(9, rot, device=dev)[9:]
    kw, vw = kp.clone(), vp.clone()
    y = paged_kv_append(q, k, v, kp, vp, tab, ctx, rope=table, interleaved=interleaved)
    for s, n in enumerate(lens):
        at = int(tab[s, (n - 1) // 16]), slice(None), (n - 1) % 16
        kw[at], vw[at] = k[s], v[s]
        kw[at][:, :rot] = float("nan")
    want = q.clone()
    want[..., :rot] = float("nan")
    for a, b in ((y, want), (kp, kw), (vp, vw)):
        assert torch.equal(a.isnan(), b.isnan()) and torch.equal(a.nan_to_num(), b.nan_to_num())


def test_layer_behind_a_prefix_as_long_as_its_table(dev):
    mods = [torch.nn.Linear(128, n, bias=False, device=dev) for n in (256, 128, 128)] + [torch.nn.Linear(256, 128, bias=False, device=dev)]
    layer = PagedAttentionLayer(*mods, head_dim=64, rope=rope_table(32, 64, device=dev))
    kp, vp, tab, ctx = cache([1, 1, 32], 2, 64, 16, FP, 36)
    y = layer(torch.randn(2, 128, device=dev), kp, vp, tab[:2], ctx[:2], prefix=(tab[2].contiguous(), 32))
    assert bool(y.isnan().all())


@pytest.mark.parametrize("dtype", [torch.int64, torch.uint32])
def test_indexes_wider_than_the_kernels(dev, dtype):
    """Ids whose low 32 bits are an id of the pool hold no tokens."""
    lens = [70, 200]
    kp, vp, tab, ctx = cache(lens, 2, 64, 16, FP, 38)
    q = _q(2, 4, 64, FP)
    wide = tab.clamp(min=0).to(torch.int64)
    wide[0, 1], wide[1, 3] = (2 ** 32 + int(tab[0, 1]), -2 ** 33 + int(tab[1, 3])) if dtype == torch.int64 else (2 ** 31 + 1, 2 ** 32 - 1)
    tab[0, 1] = tab[1, 3] = -1
    y = paged_attention(q, kp, vp, wide.to(dtype), ctx.to(dtype))
    check(y, *attention(q, kp, vp, tab, lens))


@pytest.mark.parametrize("dtype,D", [(BF, 128), (FP, 64), (HF, 80)])
@pytest.mark.parametrize("new", [[40, 5, 9], [200, 3, 130]])
@pytest.mark.parametrize("window", [2 ** 31 - 1, 2 ** 40, 2 ** 31 - 30])
def test_windows_of_any_size(dev, dtype, D, new, window):
    """Rows far below position 0 (fewer cached tokens than rows), with a window as wide as can be said."""
    lens = [25, 0, 5]
    kp, vp, tab, ctx = cache(lens, 2, D, 16, dtype, 39)
    q = _q(sum(new), 4, D, dtype)
    for pl in (None, torch.tensor([9, 3, 4], dtype=torch.int32, device=dev)):
        y = paged_attention(q, kp, vp, tab, ctx, offsets(new), window=window, prefix_lens=pl)
        check(y, *attention(q, kp, vp, tab, lens, new, window=window, prefix_lens=pl))


@pytest.mark.parametrize("window", [0, 50, 2 ** 40])
@pytest.mark.parametrize("shared", [300, 5])
def test_lengths_near_2_31_behind_a_prefix(dev, window, shared):
    """A context past its table is cut there, and its position counts as it is, also where the prefix carries it past 2^31."""
    kp, vp, tab, ctx = cache([40, 33, 2, 300], 2, 64, 16, BF, 40)
    pre, tab, ctx = tab[3, :-(-shared // 16)].contiguous(), tab[:3, :3].contiguous(), ctx[:3].clone()
    ctx[0], ctx[2] = 2 ** 31 - 1, 2 ** 31 - 200
    q = _q(3, 4, 64, BF)
    y = shared_prefix_attention(q, kp, vp, pre, shared, tab, ctx, window=window)
    check(y, *attention(q, kp, vp, tab, ctx.tolist(), shared=pre, shared_len=shared, window=window))


@pytest.mark.parametrize("dtype,D", [(BF, 128), (HF, 64), (FP, 64), (HF, 256)])
@pytest.mark.parametrize("cap", [257.0, 2e3, 1e4, 1e5, 1e6, 1e8, 9e29, 2e38])
@pytest.mark.parametrize("lens,new", [([3, 9, 70], None), ([40, 7], [40, 5]), ([300], [200])])
def test_caps_far_above_the_scores(dev, dtype, D, cap, lens, new):
    """The cap changes little then, and costs no precision: no term of the cap's size in the bound, only tanh and its two
    factors, 2^-21 of the largest score (at most the largest |q| |k| times the scale)."""
    kp, vp, tab, ctx = cache(lens, 2, D, 16, dtype, 41)
    T = sum(new) if new else len(lens)
    q = _q(T, 8, D, dtype)
    want, _ = attention(q, kp, vp, tab, lens, new, softcap=cap)
    share, bound = attention(q, kp, vp.abs(), tab, lens, new)
    score = float(q.double().norm(dim=-1).max() * kp.double().norm(dim=-1).max()) * D ** -0.5
    y = paged_attention(q, kp, vp, tab, ctx, offsets(new) if new else None, softcap=cap)
    check(y, want, bound + 2 * 2.0 ** -21 * score * share, f"{cap}")


@pytest.mark.parametrize("dtype", [BF, FP])
def test_caps_far_below_the_scores(dev, dtype):
    """All scores are the cap or its negative, and 0 where a product is 0: the mean of the values, to rounding."""
    lens = [50]
    kp, vp, tab, ctx = cache(lens, 1, 64, 16, dtype, 42)
    kp[int(tab[0, 0]), 0, 3] = 0
    q = _q(1, 4, 64, dtype)
    for cap in (1e-6, 1e-30, 1e-40):
        check(paged_attention(q, kp, vp, tab, ctx, softcap=cap), *attention(q, kp, vp, tab, lens, softcap=cap), f"{cap}")


def _spoil(vp, tab, lens, new, want, window, prefix_lens, places, shared=None, shared_len=0):
    """Puts `places` (sequence, or -1 for the shared prefix; token; element; value) into vp, and adds each value to the rows of
    `want` that see its token."""
    bs = vp.shape[2]
    for s, j, d, bad in places:
        row = shared if s < 0 else tab[s]
        vp[int(row[j // bs]), :, j % bs, d] = bad
        first = 0
        for i, (cnt, n) in enumerate(zip(new, lens)):
            if s in (i, -1):
                at = j + (shared_len if s >= 0 else 0)
                pos = torch.arange(n - cnt, n, device=vp.device).clamp(min=-1 if shared is not None else -2 ** 31) + shared_len
                sees = pos >= at
                if prefix_lens is not None:
                    sees = sees | (at < int(prefix_lens[i]))
                if window:
                    sees = sees & (pos - at < window)
                part = want[first:first + cnt, :, d]
                want[first:first + cnt, :, d] = torch.where(sees[:, None], part + torch.full_like(part, bad), part)
            first += cnt


def _check_spoilt(y, want, bound, what=""):
    y, odd = y.double(), ~torch.isfinite(want)
    assert bool((~torch.isfinite(y) == odd).all()), f"{what}: {int((~torch.isfinite(y) != odd).sum())} elements"
    assert bool(((y == want) | (y.isnan() & want.isnan()))[odd].all()), what
    check(torch.where(odd, 0.0, y), torch.where(odd, 0.0, want), torch.where(odd, 1e-30, bound), what)


INF, NAN = float("inf"), float("nan")


@pytest.mark.parametrize("dtype,D,bs", [(BF, 128, 16), (HF, 64, 8), (FP, 64, 16), (BF, 256, 16), (FP, 256, 8), (HF, 80, 24), (BF, 50, 5)])
@pytest.mark.parametrize("group", [1, 4])
@pytest.mark.parametrize("opts", ["plain", "window", "prefix", "all"])
def test_rows_apart_from_values_that_are_no_numbers(dev, dtype, D, bs, group, opts):
    """Bad values early (every row sees them), among the new tokens, at the edges of windows, of both signs in one element, in
    tokens behind a prefix mask, beside tables with holes: each reaches its element of the rows that see its token."""
    new, past = [300, 7, 70, 2], [5, 200, 0, 90]
    lens = [a + b for a, b in zip(new, past)]
    kp, vp, tab, ctx = cache(lens, 2, D, bs, dtype, 51)
    tab[2, 1] = -1
    q = _q(sum(new), 2 * group, D, dtype)
    window = 40 if opts in ("window", "all") else 0
    pl = torch.tensor([60, 205, 9, 0], dtype=torch.int32, device=dev) if opts in ("prefix", "all") else None
    o = dict(window=window, prefix_lens=pl, **(dict(softcap=5.0, slopes=torch.full((2 * group,), 0.1, device=dev)) if opts == "all" else {}))
    want, bound = attention(q, kp, vp, tab, lens, new, **o)
    _spoil(vp, tab, lens, new, want, window, pl, [
        (0, 0, 0, INF), (0, 150, 1, NAN), (0, 151, 2, INF), (0, 190, 2, -INF), (0, 304, 3, -INF), (0, 55, 4, NAN), (0, 62, 5, INF),
        (1, 202, 6, INF), (1, 206, 7, NAN), (1, 170, 8, -INF), (2, 69, 9, NAN), (2, 3 * bs, 10, INF), (3, 91, 11, NAN), (3, 0, 12, INF)])
    for hint in (None, 3, 300):
        _check_spoilt(paged_attention(q, kp, vp, tab, ctx, offsets(new), max_new=hint, **o), want, bound, f"{hint}")


@pytest.mark.parametrize("dtype,D", [(BF, 128), (FP, 64), (HF, 256)])
@pytest.mark.parametrize("n", [5, 90])
@pytest.mark.parametrize("window", [0, 130])
def test_rows_behind_a_prefix_of_values_that_are_no_numbers(dev, dtype, D, n, window):
    """Sequences of other lengths see other parts of the prefix within their windows."""
    shared = 300
    lens = [(41 * i) % 150 for i in range(n)]
    kp, vp, tab, ctx = cache(lens + [shared], 2, D, 16, dtype, 52)
    pre, tab, ctx = tab[n, :-(-shared // 16)].contiguous(), tab[:n], ctx[:n]
    q = _q(n, 8, D, dtype)
    want, bound = attention(q, kp, vp, tab, lens, shared=pre, shared_len=shared, window=window)
    _spoil(vp, tab, lens, [1] * n, want, window, None, [(-1, 200, 0, INF), (-1, 250, 1, NAN), (-1, 299, 2, -INF), (-1, 20, 3, NAN),
                                                       (-1, 280, 2, INF), (4, 0, 5, NAN), (3, 100, 6, -INF)], pre, shared)
    _check_spoilt(shared_prefix_attention(q, kp, vp, pre, shared, tab, ctx, window=window), want, bound)


@pytest.mark.parametrize("dtype,D", [(BF, 128), (FP, 64)])
@pytest.mark.parametrize("new", [[260, 3], [3, 2]])
def test_all_values_infinite(dev, dtype, D, new):
    """Every row sees infinities alone, but the rows that see nothing."""
    lens = [255, 40]
    kp, vp, tab, ctx = cache(lens, 2, D, 16, dtype, 53)
    vp.fill_(INF)
    q = _q(sum(new), 8, D, dtype)
    y = paged_attention(q, kp, vp, tab, ctx, offsets(new))
    empty = max(new[0] - lens[0], 0)
    assert bool((y[:empty] == 0).all()) and bool((y[empty:] == INF).all())


@pytest.mark.parametrize("dtype,D", [(BF, 128), (FP, 64), (HF, 80), (BF, 33), (FP, 256)])
@pytest.mark.parametrize("new,past", [([1, 1, 1], [70, 2, 400]), ([3, 2, 4], [70, 2, 400]), ([150, 1, 90], [0, 33, 200])])
def test_whole_tokens_of_no_numbers(dev, dtype, D, new, past):
    """A token whose values are all NaN: every element of the rows that see it, nothing of the others; and a cache of NaN alone."""
    lens = [a + b for a, b in zip(new, past)]
    kp, vp, tab, ctx = cache(lens, 2, D, 16, dtype, 54)
    q = _q(sum(new), 8, D, dtype)
    cu = offsets(new) if max(new) > 1 else None
    want, bound = attention(q, kp, vp, tab, lens, new)
    places = [(0, lens[0] - new[0] // 2 - 1, d, NAN) for d in range(D)] + [(2, 50, d, NAN) for d in range(D)]
    _spoil(vp, tab, lens, new, want, 0, None, places)
    _check_spoilt(paged_attention(q, kp, vp, tab, ctx, cu), want, bound)
    vp.fill_(NAN)
    assert bool(paged_attention(q, kp, vp, tab, ctx, cu).isnan().all())
