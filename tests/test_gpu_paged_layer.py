"""PagedAttentionLayer: prompts, chunks, drafted tokens, single tokens and a shared prefix through one cache give what the
whole sequences give at once. fp32: two ways of one sum differ by their roundings, and every step (projections of
up to 256 terms of 2^-24, scores, sums over 60 keys) loses less than 2^-24 of about 1000 parts of values near 1: 1e-4."""

from __future__ import annotations

import pytest
import torch
import torch.nn as nn

from serve.paged_layer import PagedAttentionLayer, rope_table

pytestmark = pytest.mark.gpu

DIM, HEADS, KV, D, BS = 256, 4, 2, 64, 16


def _layer(dtype=torch.float32, **kw):
    torch.manual_seed(0)
    mods = [nn.Linear(a, b, bias=False) for a, b in ((DIM, HEADS * D), (DIM, KV * D), (DIM, KV * D), (HEADS * D, DIM))]
    return PagedAttentionLayer(*mods, head_dim=D, rope=rope_table(128, D), **kw).to("cuda", dtype if dtype != torch.float32 else None)


def _ints(*v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


@torch.no_grad()
def _plain(layer, x):
    """One sequence, x [tokens, DIM], in 64 bits with no cache."""
    q, k, v = ((x.double() @ w.weight.double().T).unflatten(-1, (-1, D)) for w in (layer.wq, layer.wk, layer.wv))
    c, s = layer.rope[:len(x), None, :D // 2].double(), layer.rope[:len(x), None, D // 2:].double()
    turn = lambda t: torch.cat([t[..., :D // 2] * c - t[..., D // 2:] * s, t[..., :D // 2] * s + t[..., D // 2:] * c], -1)
    q, k = turn(q), turn(k)
    k, v = (t.repeat_interleave(HEADS // KV, 1) for t in (k, v))
    sc = (q.transpose(0, 1) @ k.permute(1, 2, 0).contiguous()) * D ** -0.5
    i = torch.arange(len(x), device=x.device)
    sc = sc.masked_fill(i[None, :] > i[:, None], -torch.inf)
    y = (sc.softmax(-1) @ v.transpose(0, 1).contiguous()).transpose(0, 1)
    return y.flatten(-2) @ layer.wo.weight.double().T


def _pools(n, dtype=torch.float32):
    return torch.full((2, n, KV, BS, D), float("nan"), dtype=dtype, device="cuda").unbind(0)


def test_prompt_chunk_draft_and_decode():
    layer = _layer()
    x = torch.randn(2, 60, DIM, device="cuda")
    kp, vp = _pools(12)
    tables = torch.arange(11, -1, -1, dtype=torch.int32, device="cuda").reshape(2, 6)
    out = [[], []]
    at = [0, 0]
    for new in ((17, 3), (1, 30), (16, 16), (4, 0), (1, 1)):  # prompts, a chunk beside a decode step, drafts, ..
        rows = torch.cat([x[s, at[s]:at[s] + new[s]] for s in range(2)])
        at = [a + b for a, b in zip(at, new)]
        y = layer(rows, kp, vp, tables, _ints(*at), None if new == (1, 1) else _ints(0, new[0], sum(new)))
        for s, part in enumerate(y.split(new)):
            out[s].append(part)
    for s in range(2):
        got = torch.cat(out[s])
        assert float((got.double() - _plain(layer, x[s, :len(got)])).abs().max()) < 1e-4


def test_shared_prefix():
    layer = _layer()
    common, x = torch.randn(37, DIM, device="cuda"), torch.randn(5, 3, DIM, device="cuda")
    kp, vp = _pools(8)
    shared = _ints(6, 0, 3)
    layer(common, kp, vp, shared[None], _ints(37), _ints(0, 37))
    tables = _ints(1, 2, 4, 5, 7)[:, None]
    got = torch.stack([layer(x[:, t], kp, vp, tables, torch.full((5,), t + 1, dtype=torch.int32, device="cuda"), prefix=(shared, 37))
                       for t in range(3)], 1)
    for s in range(5):
        want = _plain(layer, torch.cat([common, x[s]]))[37:]
        assert float((got[s].double() - want).abs().max()) < 1e-4
    with pytest.raises(ValueError, match="one new token a sequence"):
        layer(x[:, 0], kp, vp, tables, _ints(1, 1, 1, 1, 1), _ints(0, 1, 2, 3, 4, 5), prefix=(shared, 37))


def test_quantized_projections_and_graph():
    """A captured decode step of the INT8 layer is the eager step's, replay after replay."""
    layer = _layer(torch.bfloat16).to_int(8)
    kp, vp = _pools(8, torch.bfloat16)
    tables = torch.arange(8, dtype=torch.int32, device="cuda").reshape(4, 2)
    lens = _ints(0, 0, 0, 0)
    xs = torch.randn(20, 4, DIM, device="cuda").bfloat16()
    want = []
    for x in xs:
        lens += 1
        want.append(layer(x, kp, vp, tables, lens))
    kp.fill_(float("nan")), vp.fill_(float("nan")), lens.zero_()
    x = xs[0].clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        layer(x, kp, vp, tables, lens + 1)
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y = layer(x, kp, vp, tables, lens)
    for step, w in zip(xs, want):
        lens += 1
        x.copy_(step)
        g.replay()
        torch.cuda.synchronize()
        assert torch.isfinite(y).all() and torch.equal(y, w)
