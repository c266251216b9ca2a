"""kernels.int8_act against plain implementations in 64 bits, at the sizes, strides and values where it can go wrong.

Tolerances count roundings: u = 2^-24 is half a step of fp32 relative to the value, eps / 2 half a step of the output's type, and
`tiny` the smallest step that the type has near zero (fp32 and bf16: half of it and more)."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from kernels import int8_act as a8

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
TYPES = [F32, F16, BF16]
U = 2.0 ** -24


def half_step(t):
    return torch.finfo(t).eps / 2


def tiny(t):
    return {F32: 2.0 ** -149, F16: 2.0 ** -24, BF16: 2.0 ** -133}[t]


def gen(seed=0):
    return torch.Generator().manual_seed(seed)


def rows_like(M, K, dtype, seed=0):
    """Rows of very different sizes, one value in 16 well above the others."""
    g = gen(seed)
    x = torch.randn(M, K, generator=g) * torch.exp(2 * torch.randn(M, 1, generator=g))
    return (x * torch.where(torch.rand(M, K, generator=g) < 1 / 16, 8.0, 1.0)).to(dtype)


def codes_of(x):
    """The definition, in numpy's IEEE fp32."""
    f = x.float().numpy()
    s = np.maximum(np.abs(f).max(1) / np.float32(127), np.float32(1e-8)) if f.shape[1] else np.full(len(f), 1e-8, np.float32)
    return np.rint(f / s[:, None]).astype(np.int8), s


def weights(N, K, seed=1, dtype=F32):
    g = gen(seed)
    return (torch.randint(-127, 128, (N, K), generator=g, dtype=torch.int8).cuda(),
            (torch.rand(N, generator=g) * 0.02 + 1e-3).to(dtype).cuda())


def check_product(y, x_q, sx, w_q, sw, bias=None):
    p = (x_q.double() @ w_q.double().t()) * sw.double() * sx.double()[:, None]
    b = torch.zeros(()) if bias is None else bias.double()
    b = b.to(p.device)
    ref = p + b
    # the sum's conversion, two scales and the bias, then one rounding to the output's type
    tol = 4 * U * (p.abs() + b.abs()) * (1 + half_step(y.dtype)) + half_step(y.dtype) * ref.abs() + tiny(y.dtype)
    off = (y.double() - ref).abs()
    # from half a step past the type's largest value, max (1 + eps / 4), a number rounds to an infinity
    past = torch.isinf(y) & (y.sign() == ref.sign()) & (ref.abs() + tol >= torch.finfo(y.dtype).max * (1 + half_step(y.dtype) / 2))
    assert bool(((off <= tol) | past).all()), float((off / tol)[~past].max())


# ---------------------------------------------------------------- quantize_rows

@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M,K", [(1, 1), (3, 7), (5, 8), (2, 63), (9, 512), (4, 513), (3, 1024), (1, 1025), (2, 2048), (2, 2056), (1, 4096),
                                 (2, 8191), (1, 11008), (2, 16400), (1, 32768), (2, 33001)])
def test_codes_are_the_definition(M, K, dtype):
    x = rows_like(M, K, dtype, K)
    q, s = a8.quantize_rows(x.cuda())
    want_q, want_s = codes_of(x)
    assert q.shape == (M, K) and q.dtype == torch.int8 and s.dtype == F32
    assert np.array_equal(s.cpu().numpy(), want_s)
    assert np.array_equal(q.cpu().numpy(), want_q)


# Past 512 rows blocks hold fewer threads a row: both sides of each length at which their form changes, lengths that end inside a
# block's last columns, and of 8 but not 16.
MANY = [(513, K) for K in (1032, 2048, 2056, 4096, 4104, 5632, 6144, 6152, 8192, 8200, 11008, 12288, 12296, 16384, 16392, 32776)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M,K", MANY + [(520, 5633), (520, 11001)])
def test_codes_of_many_rows_are_the_definition(M, K, dtype):
    x = rows_like(M, K, dtype, K)
    q, s = a8.quantize_rows(x.cuda())
    want_q, want_s = codes_of(x)
    assert np.array_equal(s.cpu().numpy(), want_s)
    assert np.array_equal(q.cpu().numpy(), want_q)


@pytest.mark.parametrize("M,H", MANY + [(520, 5633), (520, 11001)])
def test_silu_mul_quantize_of_many_rows(M, H):
    """What the rows give in two calls of fewer than 512, and the checkpoint's codes by their definition."""
    dtype = TYPES[H // 8 % 3]
    gate, up = (3 * torch.randn(M, H, generator=gen(H))).to(dtype).cuda(), rows_like(M, H, dtype, H + 1).cuda()
    q, s, (kq, ks) = a8.silu_mul_quantize(gate, up, checkpoint=True)
    q2, s2 = a8.silu_mul_quantize(gate, up)
    assert torch.equal(q, q2) and torch.equal(s, s2)
    parts = [a8.silu_mul_quantize(gate[i], up[i], checkpoint=True) for i in (slice(0, 256), slice(256, M))]
    assert torch.equal(q, torch.cat([t[0] for t in parts])) and torch.equal(s, torch.cat([t[1] for t in parts]))
    G = -(-H // 128)
    for i, t in enumerate((gate, up)):
        t = torch.nn.functional.pad(t.float().cpu(), (0, G * 128 - H)).reshape(M * G, 128)
        want_q, want_s = codes_of(t)
        assert np.array_equal(ks[i].cpu().numpy(), want_s.reshape(M, G))
        assert np.array_equal(kq[i].cpu().numpy(), want_q.reshape(M, G * 128)[:, :H])


@pytest.mark.parametrize("K", [8, 1032])
def test_more_rows_than_a_launch(K):
    """2^21 rows and some: those at both ends and around the second launch's first are what they are in a call of their own."""
    M = 2 ** 21 + 5
    x = torch.randn(M, K, device="cuda", dtype=BF16, generator=torch.Generator("cuda").manual_seed(1))
    q, s = a8.quantize_rows(x)
    h_q, h_s, (kq, ks) = a8.silu_mul_quantize(x, x, checkpoint=True)
    for r in (slice(0, 9), slice(2 ** 21 - 9, 2 ** 21), slice(2 ** 21, M)):
        a, (b, c, (d, e)) = a8.quantize_rows(x[r]), a8.silu_mul_quantize(x[r], x[r], checkpoint=True)
        for got, want in ((q[r], a[0]), (s[r], a[1]), (h_q[r], b), (h_s[r], c), (kq[:, r], d), (ks[:, r], e)):
            assert torch.equal(got, want)


def test_codes_next_to_ties_and_of_every_size():
    """Quotients at and beside every tie, and rows from 1e-45 to 3e38."""
    g = gen(3)
    s = torch.exp(torch.empty(400, 1).uniform_(-18, 80, generator=g))
    k = torch.arange(-127, 127) + 0.5
    x = (s.double() * k.double()).float()
    x = torch.cat([x, torch.nextafter(x, torch.full_like(x, torch.inf)), torch.nextafter(x, torch.zeros(()).expand_as(x))], 1)
    x = torch.cat([x, s * 127], 1)
    top = torch.tensor([[1e-45, -1e-45], [1e-8, 3e-9], [1.27e-6, 1e-6], [3.4e38, -3.4e38], [0.0, -0.0]])
    for t in (x, top):
        q, sc = a8.quantize_rows(t.cuda())
        want_q, want_s = codes_of(t)
        assert np.array_equal(sc.cpu().numpy(), want_s) and np.array_equal(q.cpu().numpy(), want_q)


def test_codes_agree_with_the_weight_quantizer():
    from serve.quantize import quantize_int8
    w = rows_like(33, 777, F32).cuda()
    q, s = a8.quantize_rows(w)
    wq, ws = quantize_int8(w)
    assert torch.equal(q, wq) and torch.equal(s, ws)


@pytest.mark.parametrize("bad", [float("inf"), -float("inf"), float("nan")])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M", [3, 40])
def test_a_value_that_is_no_number_stays_in_its_row(M, dtype, bad):
    x = rows_like(M, 300, dtype)
    x[1, 77] = bad
    q, s = a8.quantize_rows(x.cuda())
    want_q, want_s = codes_of(x[[0, 2]])
    assert not bool(torch.isfinite(s[1])) and not bool(q[1].any())
    assert np.array_equal(q[[0, 2]].cpu().numpy(), want_q) and np.array_equal(s[[0, 2]].cpu().numpy(), want_s)
    w_q, sw = weights(50, 300)
    y = a8.int8_dynamic_matmul(x.cuda(), w_q, sw)
    assert bool(torch.isnan(y[1]).all()) and bool(torch.isfinite(y[[0, 2]]).all())


@pytest.mark.parametrize("M", [1, 5, 40])
def test_strided_inputs(M):
    """Rows apart, starting at odd places, expanded, transposed: the same as their dense copies."""
    base = rows_like(M, 700, BF16).cuda()
    w_q, sw = weights(70, 333)
    big = torch.zeros(70, 400, dtype=torch.int8, device="cuda")
    big[:, 5:338] = w_q
    for x in (base[:, 1:334], base[:, 300:633], base.t().contiguous().t()[:, :333], base[:1, :333].expand(M, 333)):
        q, s = a8.quantize_rows(x)
        qc, sc = a8.quantize_rows(x.contiguous())
        assert torch.equal(q, qc) and torch.equal(s, sc)
        y = a8.int8_dynamic_matmul(x.contiguous(), w_q, sw)
        for w in (big[:, 5:338], w_q.t().contiguous().t()):
            assert torch.equal(a8.int8_dynamic_matmul(x, w, sw), y)
            assert torch.equal(a8.int8_scaled_matmul(q, s, w, sw), y)
            assert torch.equal(a8.int8_scaled_matmul(qc.contiguous(), s, w, sw), y)


# ---------------------------------------------------------------- products

@pytest.mark.parametrize("M", [1, 2, 3, 8, 13, 16, 17, 31, 64, 65, 128, 129, 300])
@pytest.mark.parametrize("N,K", [(1, 1), (15, 16), (16, 100), (33, 128), (130, 272), (257, 777), (1000, 1024), (64, 4112), (48, 12000)])
def test_product(M, N, K):
    dtype = TYPES[(M + N) % 3]
    x = rows_like(M, K, dtype, M)
    w_q, sw = weights(N, K, N, F16 if K % 3 else F32)
    bias = torch.randn(N, generator=gen(5)).to(TYPES[K % 3]).cuda() if M % 2 else None
    q, s = a8.quantize_rows(x.cuda())
    check_product(a8.int8_scaled_matmul(q, s, w_q, sw, bias, out_dtype=dtype), q, s, w_q, sw, bias)
    y = a8.int8_dynamic_matmul(x.cuda(), w_q, sw, bias)
    assert y.dtype == dtype and torch.equal(y, a8.int8_scaled_matmul(q, s, w_q, sw, bias, out_dtype=dtype))


@pytest.mark.parametrize("M,N,K", [(513, 4200, 512), (700, 8192, 1280), (2049, 2100, 272), (4096, 4096, 128)])
def test_product_of_many_tiles(M, N, K):
    q, s = a8.quantize_rows(rows_like(M, K, BF16).cuda())
    w_q, sw = weights(N, K)
    for dt in TYPES:
        check_product(a8.int8_scaled_matmul(q, s, w_q, sw, out_dtype=dt), q, s, w_q, sw)


@pytest.mark.parametrize("M", [1, 16, 20, 200])
def test_sums_at_the_ends_of_32_bits(M):
    """-128 by -128 over the longest K: 2147467264, and its negative by 127 and -128."""
    K = a8.MAX_K
    x = torch.full((M, K), -128, dtype=torch.int8, device="cuda")
    w = torch.full((3, K), -128, dtype=torch.int8, device="cuda")
    w[1] = 127
    w[2, ::2] = 127
    one = torch.ones(M, device="cuda")
    y = a8.int8_scaled_matmul(x, one, w, one.new_ones(3), out_dtype=F32)
    want = torch.tensor([128 * 128 * K, -128 * 127 * K, 128 * 128 * (K // 2) - 128 * 127 * (K - K // 2)], dtype=torch.int64).float()
    assert torch.equal(y, want.cuda().expand(M, 3))


def test_scales_at_the_ends_of_fp32():
    """Rows near 3e38 and weights' scales near 1e-38: no product on the way leaves fp32."""
    q = torch.tensor([[127, 0], [1, 1], [0, 0]], dtype=torch.int8, device="cuda")
    sx = torch.tensor([2.6e36, 1e-8, 2.6e36], device="cuda")
    w = torch.tensor([[127, 3], [2, -5]], dtype=torch.int8, device="cuda")
    for sw in (torch.tensor([1e-30, 1e-8], device="cuda"), torch.tensor([1e-3, 1e3], device="cuda")):
        y = a8.int8_scaled_matmul(q, sx, w, sw, out_dtype=F32)
        ref = ((q.double() @ w.double().t()) * sw.double() * sx.double()[:, None])
        fits = ref.abs() < 3.4e38
        assert bool(torch.isfinite(y[fits]).all()) and torch.allclose(y[fits].double(), ref[fits], rtol=4 * U, atol=0)


def test_sizes_of_zero():
    w_q, sw = weights(5, 32)
    bias = torch.randn(5, device="cuda")
    assert a8.int8_dynamic_matmul(torch.zeros(0, 32, device="cuda"), w_q, sw).shape == (0, 5)
    assert a8.int8_dynamic_matmul(torch.ones(3, 32, device="cuda"), w_q[:0], sw[:0]).shape == (3, 0)
    y = a8.int8_dynamic_matmul(torch.ones(3, 0, device="cuda"), w_q[:, :0], sw, bias)
    assert torch.equal(y, bias.expand(3, 5))
    assert not a8.int8_dynamic_matmul(torch.ones(3, 0, device="cuda"), w_q[:, :0], sw).any()
    q, s = a8.quantize_rows(torch.zeros(2, 0, device="cuda"))
    assert q.shape == (2, 0) and torch.equal(s, torch.full_like(s, 1e-8))
    assert a8.quantize_rows(torch.zeros(0, 9, device="cuda"))[0].shape == (0, 9)
    for M, H in ((0, 40), (3, 0)):
        z = torch.zeros(M, H, device="cuda")
        q, s, kept = a8.silu_mul_quantize(z, z, checkpoint=True)
        assert q.shape == (M, H) and s.shape == (M,) and kept[0].shape == (2, M, H)
        dg, du = a8.silu_mul_backward(z, kept)
        assert dg.shape == du.shape == (M, H)
    dw = a8.int8_weight_grad(torch.zeros(0, 4, device="cuda"), torch.zeros(0, 6, dtype=torch.int8, device="cuda"), torch.zeros(0, device="cuda"))
    assert dw.shape == (4, 6) and not dw.any()
    assert a8.int8_weight_grad(torch.zeros(3, 0, device="cuda"), torch.zeros(3, 6, dtype=torch.int8, device="cuda"), torch.zeros(3, device="cuda")).shape == (0, 6)


@pytest.mark.parametrize("M", [1, 16, 40, 300])
def test_rows_behind_the_operands_are_not_read(M):
    """Operands inside larger buffers whose other bytes are -128 and whose other scales are NaN, K no multiple of 128."""
    K, N = 208, 70
    q, s = a8.quantize_rows(rows_like(M, K, F32, M).cuda())
    w, sw = weights(N, K)
    def inside(t, fill, rows, cols):
        big = torch.full((t.shape[0] + 2 * rows, t.shape[1] + 2 * cols), fill, dtype=t.dtype, device="cuda")
        view = big[rows:-rows, cols:t.shape[1] + cols]
        view.copy_(t)
        return view
    want = a8.int8_scaled_matmul(q, s, w, sw, out_dtype=F32)
    for cols in (16, 3):
        assert torch.equal(a8.int8_scaled_matmul(inside(q, -128, 2, cols), s, inside(w, -128, 2, cols), sw, out_dtype=F32), want)
    y = torch.full((M + 2, N + 8), 7.0, device="cuda")  # the C entry's rows of any distance: what is beside them stays
    args = a8._ARGS.pack(q.data_ptr(), s.data_ptr(), w.data_ptr(), sw.data_ptr(), 0, y[1:, 4:].data_ptr(), -1, 0, 0, 0, q.stride(0), K, N + 8, M, N, K)
    ws = torch.empty(max(1, a8.kernels.lib().mlsx_a8w8_ws(args)), dtype=torch.uint8, device="cuda")
    assert a8.kernels.lib().mlsx_a8w8(args, ws.data_ptr(), ws.numel(), torch.cuda.current_stream().cuda_stream) == 0
    assert torch.equal(y[1:-1, 4:-4], want)
    y[1:-1, 4:-4] = 7.0
    assert bool((y == 7.0).all())


# ---------------------------------------------------------------- silu_mul_quantize

def sigmoid_error(g):
    """Relative error of silu(g) * u in fp32: the exponent's product off by 1.5 |g| u, the exponential and the reciprocal by a step
    (2 u) each, the sum, the two products and log2 e's own rounding by u each."""
    return (1.5 * g.abs() + 8) * U


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M,H", [(1, 1), (3, 127), (2, 128), (5, 129), (9, 1000), (4, 1024), (2, 2049), (3, 5632), (1, 11008), (2, 16500), (2, 33000)])
def test_silu_mul_quantize(M, H, dtype):
    gate, up = (3 * torch.randn(M, H, generator=gen(H))).to(dtype), rows_like(M, H, dtype, H + 1)
    q, s, (kq, ks) = a8.silu_mul_quantize(gate.cuda(), up.cuda(), checkpoint=True)
    q2, s2 = a8.silu_mul_quantize(gate.cuda(), up.cuda())
    assert torch.equal(q, q2) and torch.equal(s, s2)
    g, u = gate.double(), up.double()
    h = g * torch.sigmoid(g) * u
    e = sigmoid_error(g)
    top = h.abs().amax(1)
    err = (e * h.abs()).amax(1)  # of any value of the row
    s, q = s.double().cpu(), q.double().cpu()
    assert bool(((s - (top / 127).clamp(min=1e-8)).abs() <= err / 127 + 2 * U * s).all())
    # a code is the nearest whole number of a quotient that is off by its value's error and a rounding
    assert bool(((q - h / s[:, None]).abs() <= 0.5 + e * (h / s[:, None]).abs() + 128 * U).all())
    G = -(-H // 128)
    for i, t in enumerate((gate, up)):
        t = torch.nn.functional.pad(t.float(), (0, G * 128 - H)).reshape(M * G, 128)
        want_q, want_s = codes_of(t)
        assert np.array_equal(ks[i].cpu().numpy(), want_s.reshape(M, G))
        assert np.array_equal(kq[i].cpu().numpy(), want_q.reshape(M, G * 128)[:, :H])


def test_silu_mul_quantize_strided_and_not_finite():
    both = rows_like(7, 2 * 300 + 1, BF16).cuda()
    gate, up = both[:, 1:301], both[:, 301:]
    a = a8.silu_mul_quantize(gate, up, checkpoint=True)
    b = a8.silu_mul_quantize(gate.contiguous(), up.contiguous(), checkpoint=True)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1]) and torch.equal(a[2][0], b[2][0]) and torch.equal(a[2][1], b[2][1])
    gate, up = gate.clone(), up.clone()
    gate[2, 140] = float("nan")
    up[3, 5] = float("inf")
    q, s, kept = a8.silu_mul_quantize(gate, up, checkpoint=True)
    keep = [0, 1, 4, 5, 6]
    assert torch.equal(q[keep], a[0][keep]) and torch.equal(s[keep], a[1][keep])
    assert not bool(torch.isfinite(s[[2, 3]]).any()) and not bool(q[[2, 3]].any())
    dg, du = a8.silu_mul_backward(torch.ones_like(gate), kept)
    assert bool(torch.isfinite(dg[keep]).all() and torch.isfinite(du[keep]).all())
    assert bool(torch.isnan(dg[2, 128:256]).all()) and bool(torch.isfinite(dg[2, :128]).all())
    big = torch.tensor([[-200.0, -90.0, 100.0, 0.0]], device="cuda")  # e^-g past fp32, and none
    q, s = a8.silu_mul_quantize(big, torch.ones_like(big))
    assert torch.equal(s, torch.full_like(s, 100 / 127)) and q.tolist() == [[0, 0, 127, 0]]


# ---------------------------------------------------------------- silu_mul_backward

@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M,H", [(1, 1), (3, 127), (2, 128), (5, 129), (9, 1000), (40, 1365), (3, 5632)])
def test_silu_mul_backward(M, H, dtype):
    gate, up = 3 * torch.randn(M, H, generator=gen(H)), rows_like(M, H, F32, H + 1)
    _, _, (kq, ks) = a8.silu_mul_quantize(gate.cuda(), up.cuda(), checkpoint=True)
    dh = torch.randn(M, H, generator=gen(7)).to(dtype).cuda()
    wide = torch.zeros(M, H + 3, dtype=dtype, device="cuda")
    wide[:, 1:H + 1] = dh
    for d, kept in ((dh, (kq, ks)), (wide[:, 1:H + 1], (torch.cat([kq, kq], 2)[..., :H], torch.cat([ks, ks], 2)[..., :ks.shape[2]]))):
        dg, du = a8.silu_mul_backward(d, kept)
        g, u = (kq.double() * ks.double().repeat_interleave(128, 2)[..., :H])
        sig = torch.sigmoid(g)
        want_u = dh.double() * g * sig
        want_g = dh.double() * u * sig * (1 + g * (1 - sig))
        # sig as above; g (1 - sig) is off by |g| times sig's error and its own roundings, of a sum that can cancel
        e = sigmoid_error(g) + 3 * U
        off_u, off_g = (du.double() - want_u).abs(), (dg.double() - want_g).abs()
        assert bool((off_u <= want_u.abs() * (e + half_step(dtype)) + tiny(dtype)).all())
        whole = (dh.double() * u * sig).abs()
        assert bool((off_g <= whole * (1 + g.abs()) * (2 * e + 4 * U) + half_step(dtype) * want_g.abs() + tiny(dtype)).all())


def test_silu_mul_backward_is_the_slope():
    """Against differences of the formula in 64 bits, at the 8-bit values (step 1e-6: off by its square and the subtraction)."""
    gate, up = torch.linspace(-9, 9, 512).reshape(2, 256), rows_like(2, 256, F32)
    _, _, kept = a8.silu_mul_quantize(gate.cuda(), up.cuda(), checkpoint=True)
    dh = torch.randn(2, 256, generator=gen(2)).cuda()
    dg, du = a8.silu_mul_backward(dh, kept)
    g, u = (kept[0].double() * kept[1].double().repeat_interleave(128, 2))
    f = lambda g, u: g * torch.sigmoid(g) * u
    h = 1e-6
    scale = (1 + u.abs()) * (1 + g.abs()) * dh.abs()
    assert bool(((dg - dh * (f(g + h, u) - f(g - h, u)) / (2 * h)).abs() <= 1e-5 * scale).all())
    assert bool(((du - dh * (f(g, u + h) - f(g, u - h)) / (2 * h)).abs() <= 1e-5 * scale).all())


# ---------------------------------------------------------------- int8_weight_grad

def check_dw(dw, dy, q, s):
    ref = dy.double().t() @ (q.double() * s.double()[:, None])
    size = dy.double().abs().t() @ (q.double().abs() * s.double()[:, None])
    # the kept value's rounding to dy's type (fp32: its product's), and an fp32 rounding or truncation (2 u) a term of the sum
    tol = size * (half_step(dw.dtype) + (2 * len(dy) + 16) * U) + half_step(dw.dtype) * ref.abs() + tiny(dw.dtype) * (1 + dy.double().abs().sum(0)[:, None])
    off = (dw.double() - ref).abs()
    assert bool((off <= tol).all()), float((off / tol).max())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M,N,K", [(1, 1, 1), (2, 3, 5), (7, 16, 16), (31, 100, 33), (64, 128, 128), (65, 129, 257), (200, 64, 1000), (777, 300, 130),
                                   (1030, 40, 24)])
def test_weight_grad(M, N, K, dtype):
    q, s = a8.quantize_rows(rows_like(M, K, dtype, M).cuda())
    dy = (torch.randn(M, N, generator=gen(M)) * 0.1).to(dtype).cuda()
    dw = a8.int8_weight_grad(dy, q, s)
    assert dw.dtype == dtype and dw.shape == (N, K)
    check_dw(dw, dy, q, s)
    wide = torch.full((M, N + 5), float("nan"), dtype=dtype, device="cuda")
    wide[:, 3:N + 3] = dy
    assert torch.equal(a8.int8_weight_grad(wide[:, 3:N + 3], q.contiguous(), s), dw)
    assert torch.equal(a8.int8_weight_grad(dy.t().contiguous().t(), q.t().contiguous().t(), s), dw)


@pytest.mark.parametrize("dtype,M,N,K", [(BF16, 130, 4100, 2900), (F16, 333, 2900, 4100), (F32, 300, 1500, 1100)])
def test_weight_grad_of_many_tiles(dtype, M, N, K):
    q, s = a8.quantize_rows(rows_like(M, K, dtype, M).cuda())
    dy = (torch.randn(M, N, generator=gen(M)) * 0.1).to(dtype).cuda()
    check_dw(a8.int8_weight_grad(dy, q, s), dy, q, s)


@pytest.mark.parametrize("dtype", TYPES)
def test_weight_grad_keeps_nan_and_infinity_where_they_are(dtype):
    q, s = a8.quantize_rows(rows_like(100, 40, dtype).cuda())
    dy = torch.randn(100, 30, generator=gen(1)).to(dtype).cuda()
    dy[50, 7] = float("nan")
    dy[3, 20] = float("inf")
    dw = a8.int8_weight_grad(dy, q, s)
    assert bool(torch.isnan(dw[7]).all()) and not bool(torch.isfinite(dw[20]).any())
    keep = [i for i in range(30) if i not in (7, 20)]
    check_dw(dw[keep], dy[:, keep], q, s)


# ---------------------------------------------------------------- streams and graphs

def a_run(x, gate, up, dy, dh, w, wd):
    """Every operator once, as a layer would."""
    y = a8.int8_dynamic_matmul(x, *w)
    q, s, kept = a8.silu_mul_quantize(gate, up, checkpoint=True)
    z = a8.int8_scaled_matmul(q, s, *wd, out_dtype=x.dtype)
    return [y, z, *a8.silu_mul_backward(dh, kept), a8.int8_weight_grad(dy, q, s)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M", [1, 9, 150])
def test_replayed_graphs(M, dtype):
    """A captured run replayed over new inputs, with eager runs and synchronizations between the replays."""
    K, H, N = 300, 520, 260
    w, wd = weights(H, K), weights(N, H)
    make = lambda i: [rows_like(M, n, dtype, 9 * i + j).cuda() for j, n in enumerate((K, H, H, N, H))]
    static = make(0)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        a_run(*static, w, wd)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = a_run(*static, w, wd)
    for i in range(1, 5):
        new = make(i)
        for a, b in zip(static, new):
            a.copy_(b)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(out, a_run(*new, w, wd)):
            assert torch.equal(a, b)


def test_another_stream():
    x = rows_like(150, 512, BF16).cuda()
    w_q, sw = weights(256, 512)
    want = a8.int8_dynamic_matmul(x, w_q, sw)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        late = torch.zeros_like(x)
        for _ in range(20):  # work in front of the call, on its stream
            late.copy_(x)
        y = a8.int8_dynamic_matmul(late, w_q, sw)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(y, want)
