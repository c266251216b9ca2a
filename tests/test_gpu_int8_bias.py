"""kernels.int8_act.bias_grad against sums in 64 bits."""

from __future__ import annotations

import pytest
import torch

from kernels import int8_act as a8

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
TYPES = [F32, F16, BF16]
U = 2.0 ** -24


def gen(seed):
    return torch.Generator("cuda").manual_seed(seed)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M,N", [(1, 1), (3, 7), (64, 64), (65, 130), (300, 8), (1000, 257), (8191, 40), (8193, 33), (20000, 9)])
def test_sums(M, N, dtype):
    """A rounding of 2^-24 an addition, M at most, then one to the output's type; strided and transposed rows give the same bits."""
    dy = (0.1 * torch.randn(M, N, device="cuda", generator=gen(M))).to(dtype)
    ref, size = dy.double().sum(0), dy.double().abs().sum(0)
    wide = torch.full((M, N + 5), float("nan"), dtype=dtype, device="cuda")
    wide[:, 3:N + 3] = dy
    for out in TYPES:
        db = a8.bias_grad(dy, out_dtype=out)
        half, low = torch.finfo(out).eps / 2, {F32: 2.0 ** -149, F16: 2.0 ** -25, BF16: 2.0 ** -133}[out]
        assert db.dtype == out and db.shape == (N,)
        assert bool(((db.double() - ref).abs() <= M * U * size * (1 + half) + half * ref.abs() + low).all())
        assert torch.equal(a8.bias_grad(wide[:, 3:N + 3], out_dtype=out), db) and torch.equal(a8.bias_grad(dy.t().contiguous().t(), out_dtype=out), db)
    assert a8.bias_grad(dy).dtype == dtype


@pytest.mark.parametrize("dtype", TYPES)
def test_every_row_counts_once(dtype):
    """Whole numbers whose sums are exact."""
    for M in (1, 63, 64, 65, 127, 128, 129, 4096, 8192, 8200, 12345):
        dy = torch.randint(-8, 9, (M, 70), device="cuda", generator=gen(M)).to(dtype)
        assert torch.equal(a8.bias_grad(dy, out_dtype=F32), dy.double().sum(0).float())


def test_no_numbers_and_sizes_of_zero():
    dy = torch.randn(300, 70, device="cuda", generator=gen(1))
    dy[299, 3], dy[0, 68] = float("nan"), float("inf")
    db = a8.bias_grad(dy)
    keep = [n for n in range(70) if n not in (3, 68)]
    assert bool(torch.isnan(db[3])) and bool(torch.isinf(db[68])) and bool(torch.isfinite(db[keep]).all())
    assert torch.equal(a8.bias_grad(torch.zeros(0, 5, device="cuda")), torch.zeros(5, device="cuda"))
    assert a8.bias_grad(torch.zeros(4, 0, device="cuda")).shape == (0,)


@pytest.mark.parametrize("M", [40, 1000])
def test_replayed(M):
    static = torch.zeros(M, 130, device="cuda", dtype=BF16)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        a8.bias_grad(static)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = a8.bias_grad(static)
    for i in range(4):
        new = torch.randn(M, 130, device="cuda", generator=gen(i)).to(BF16)
        static.copy_(new)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, a8.bias_grad(new))
