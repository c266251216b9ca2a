"""Every form of tile that kernels.int8_act's products choose between, whole and in ranges of K, at sizes that the rule itself sends there.

The numbers are such that every sum is exact in fp32, so results have to be equal to those of 64 bits."""

from __future__ import annotations

import functools
import itertools

import pytest
import torch

import kernels
from kernels import int8_act as a8

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
TYPES = [F32, F16, BF16]
CODE = {F32: kernels.MLS_F32, F16: kernels.MLS_F16, BF16: kernels.MLS_BF16}
SIZES = (17, 40, 65, 100, 131, 200, 257, 300, 333, 401, 513, 600, 701, 900, 1030, 1500, 2061, 3001, 4101, 5201)
FORMS = ["64x64", "128x64", "128x128", "128x128 in phases", "256x256"]
CASES = [(f, r) for f in range(5) for r in ((False, True) if f < 3 else (False,))]


def a8_form(M, N, K):
    ld = -(-K // 16) * 16
    return kernels.lib().mlsx_a8w8_form(a8._ARGS.pack(1 << 20, 1 << 20, 1 << 20, 1 << 20, 0, 1 << 20, -1, 0, 0, 2, ld, ld, N, M, N, K))


@functools.lru_cache(None)
def sizes_of(kind):
    """(form, in ranges, more columns than a block of the join, many stages) -> the smallest rows, columns, length that the rule sends there."""
    ask = a8_form if kind == "a8" else lambda R, C, L: kernels.lib().mlsx_dw_int8_form(kind, L, R, C)
    lengths = (131, 272, 777, 1040, 2061, 4112, 8208) if kind == "a8" else (65, 130, 300, 701, 1030, 2100, 4100)
    found = {}
    for s in itertools.product(SIZES[:17], SIZES, lengths):
        code = ask(*s)
        key = code // 16 - 1, code % 16 > 1, s[1] > 1024, s[2] >= 1030
        if key not in found or s[0] * s[1] * s[2] < found[key][0]:
            found[key] = s[0] * s[1] * s[2], s
    return {k: v[1] for k, v in found.items()}


def picked(kind, form, ranges):
    """Those sizes: of few columns and of many, short and long, where the rule has them."""
    found = sizes_of(kind)
    got = [s for k, s in found.items() if k[:2] == (form, ranges)]
    assert got, f"no size in the list reaches {FORMS[form]}, ranges {ranges}"
    assert any(s[2] >= 1030 for s in got) and (not ranges or any(s[1] > 1024 for s in got))
    return got


def ints(lo, hi, *shape, seed, dtype):
    return torch.randint(lo, hi + 1, shape, device="cuda", generator=torch.Generator("cuda").manual_seed(seed)).to(dtype)


@pytest.mark.parametrize("form,ranges", CASES)
def test_product(form, ranges):
    """Codes up to 7: sums below 2^24. Scales and bias are such that their products and sums are exact too."""
    for M, N, K in picked("a8", form, ranges):
        q, w = ints(-7, 7, M, K, seed=1, dtype=torch.int8), ints(-7, 7, N, K, seed=2, dtype=torch.int8)
        sx, sw = torch.exp2(ints(-3, 3, M, seed=3, dtype=F32)), torch.exp2(ints(-3, 3, N, seed=4, dtype=F32))
        bias = ints(-8, 8, N, seed=5, dtype=F32)
        sums = q.double() @ w.double().t()
        one = torch.ones(M, device="cuda")
        for dt in TYPES:
            assert torch.equal(a8.int8_scaled_matmul(q, one, w, one.new_ones(N), out_dtype=dt), sums.float().to(dt))
        y = a8.int8_scaled_matmul(q, sx, w, sw, bias, out_dtype=F32)
        assert torch.equal(y, (sums * sx.double()[:, None] * sw.double() + bias.double()).float())
        # a K range that is left out or met twice cannot hide: one product in a row, at every place of K in turn
        q.zero_()
        at = torch.arange(M, device="cuda") * 7919 % K
        q[torch.arange(M, device="cuda"), at] = 1
        assert torch.equal(a8.int8_scaled_matmul(q, one, w, one.new_ones(N), out_dtype=F32), w.t()[at].float())


@pytest.mark.parametrize("form,ranges", CASES)
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_weight_grad_16_bit(form, ranges, dtype):
    """dy up to 8, codes of 7 bits and scales of powers of two: factors that 16-bit types hold, sums below 2^24."""
    for N, K, M in picked(CODE[dtype], form, ranges):
        q, dy = ints(-127, 127, M, K, seed=1, dtype=torch.int8), ints(-8, 8, M, N, seed=2, dtype=dtype)
        s = torch.exp2(ints(-1, 0, M, seed=3, dtype=F32))
        ref = dy.double().t() @ (q.double() * s.double()[:, None])
        for out in TYPES:
            assert torch.equal(a8.int8_weight_grad(dy, q, s, out_dtype=out), ref.float().to(out))


@pytest.mark.parametrize("form,ranges", CASES)
def test_weight_grad_fp32_is_exact(form, ranges):
    """One token in each column of dy, an odd number of 24 bits, with codes and scales that are powers of two: all three parts have to arrive, each once."""
    for N, K, M in picked(CODE[F32], form, ranges):
        n = torch.arange(N, device="cuda")
        m = n * 7919 % M
        dy = torch.zeros(M, N, device="cuda")
        dy[m, n] = (2 * ints(2 ** 22, 2 ** 23 - 1, N, seed=1, dtype=F32) + 1) * (1 - 2 * ints(0, 1, N, seed=2, dtype=F32))
        q = (ints(-1, 1, M, K, seed=3, dtype=torch.int8) * torch.exp2(ints(0, 6, M, 1, seed=4, dtype=F32))).to(torch.int8)
        s = torch.exp2(ints(-3, 3, M, seed=5, dtype=F32))
        want = dy[m, n][:, None] * (q[m].float() * s[m][:, None])
        for out in TYPES:
            assert torch.equal(a8.int8_weight_grad(dy, q, s, out_dtype=out), want.to(out))


@pytest.mark.parametrize("form,ranges", CASES)
def test_weight_grad_fp32_of_ordinary_numbers(form, ranges):
    """dy s is rounded once, and a sum has a rounding of 2^-24 for every 32 products of each part, at most 390 here: off by 390^(1/2) 2^-24
    = 1.2e-6 of the norm where they fall at random, as they do for these; 2e-6 is far below the third part's 2^-17."""
    for N, K, M in picked(CODE[F32], form, ranges):
        g = torch.Generator("cuda").manual_seed(1)
        q, dy, s = ints(-127, 127, M, K, seed=2, dtype=torch.int8), torch.randn(M, N, device="cuda", generator=g), torch.rand(M, device="cuda", generator=g) + 0.1
        ref = dy.double().t() @ (q.double() * s.double()[:, None])
        assert float((a8.int8_weight_grad(dy, q, s).double() - ref).norm()) <= 2e-6 * float(ref.norm())


def test_few_rows_say_what_they_run():
    """Up to 16 rows: no tiles, and from values the row is quantized on the way where that is short."""
    assert [a8_form(m, 64, 256) for m in (1, 16)] == [0, 0] and a8_form(17, 64, 256) >= 16
    values = lambda m, n, k: kernels.lib().mlsx_a8w8_form(a8._ARGS.pack(1 << 20, 0, 1 << 20, 1 << 20, 0, 1 << 20, 2, 0, 0, 2, k, k, n, m, n, k))
    assert values(1, 4096, 4096) == 1 and values(16, 11008, 4096) == 0
    assert kernels.lib().mlsx_a8w8_form(None) == -1 and kernels.lib().mlsx_dw_int8_form(9, 64, 64, 64) == -1 and kernels.lib().mlsx_dw_int8_form(0, 0, 64, 64) == -1


@pytest.mark.parametrize("dtype", TYPES)
def test_weight_grad_of_the_most_tokens(dtype):
    """2^20 tokens, 300 columns against 270: rows of turned operands up to 6 MiB apart. Sums of whole numbers below 2^24."""
    M, N, K = 2 ** 20, 300, 270
    q, dy = ints(-1, 1, M, K, seed=1, dtype=torch.int8), ints(-2, 2, M, N, seed=2, dtype=dtype)
    s = torch.exp2(ints(-1, 1, M, seed=3, dtype=F32))
    want = torch.zeros(N, K, dtype=torch.float64, device="cuda")
    for m in range(0, M, 2 ** 17):
        part = slice(m, m + 2 ** 17)
        want += dy[part].double().t() @ (q[part].double() * s[part].double()[:, None])
    assert torch.equal(a8.int8_weight_grad(dy, q, s, out_dtype=F32), want.float())
    with pytest.raises(NotImplementedError):
        a8.int8_weight_grad(dy[:1].expand(M + 1, N), q[:1].expand(M + 1, K), s[:1].expand(M + 1))
