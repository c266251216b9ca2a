// Activations in 8 bits: codes of rows for the int8 product, SwiGLU's product with its codes and the 8-bit
// checkpoint of its two inputs, and its backward pass from that checkpoint. All are bound by memory: 2048 x 5632 bf16 gates and
// ups with their checkpoint 20.5 us (3.9 TB/s; 21 from cold memory), the backward of 4096 x 11008 73 us (5.0 TB/s, a copy's rate).
//
// Forward kernels: a row's values stay in registers between the pass that finds its largest and the one that makes codes, so every
// input is read once. A row belongs to one wavefront (up to 1024 columns) or one block; the longest rows are read
// twice, the second time from L2.
#include "act8.h"

namespace mls {

namespace {

struct RowArgs {
  const void* x;   // quantize: the rows; silu: gate
  const void* u;   // up
  int64_t ldx, ldu;
  int64_t M, K, kpad;
  int64_t first;   // a launch's first row
  int8_t* q;
  int64_t ldq;
  float* s;
  int8_t* kept_q;  // [2][M][K]
  float* kept_s;   // [2][M][groups]
  int64_t groups;
};

// n <= 8 codes to a row, any alignment
__device__ __forceinline__ void store_codes(int8_t* dst, const uint2& c, int64_t n) {
  if (n >= 8) {
    __builtin_memcpy(dst, &c, 8);
  } else {
    const uint64_t both = (uint64_t)c.y << 32 | c.x;
    for (int e = 0; e < n; ++e) dst[e] = (int8_t)(both >> (8 * e));
  }
}

// The same of two chunks of a lane at columns ka and kb, the lanes' neighbours 8 columns on, n a multiple of 16: lanes 2 i and
// 2 i + 1 trade a chunk, so that each stores 16 bytes of one. Against stores of 8 bytes and no form of three chunks, with the checkpoint:
// 4096 x 11008 76.8 -> 64.2 us, 2048 x 5632 21.3 -> 20.5, 4096 x 8192 equal; alone, in replayed graphs, one row of
// 11008 5.7 -> 5.8 with the checkpoint and 3.6 either way without, 512 rows 13.1 -> 12.6.
__device__ __forceinline__ void store_two(int8_t* row, const uint2& a, const uint2& b, int64_t ka, int64_t kb, int64_t n, int t) {
  auto neighbour = [](uint32_t v) { return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0xB1, 0xF, 0xF, false); };
  const bool odd = t & 1;
  const uint32_t x = neighbour(odd ? a.x : b.x), y = neighbour(odd ? a.y : b.y);
  const uint4 o = odd ? make_uint4(x, y, b.x, b.y) : make_uint4(a.x, a.y, x, y);
  const int64_t k = odd ? kb - 8 : ka;
  if (k < n) __builtin_memcpy(row + k, &o, 16);
}

// The checkpoint's codes of 8 values of gate or up at column k, their scale stored: the 16 lanes of a group of 128 columns meet.
__device__ __forceinline__ uint2 keep8(const RowArgs& p, int which, int64_t m, int64_t k, const float (&v)[8]) {
  const Scale8 g = scale8(group_max_bits<16>(max_abs8(v)));
  if (k < p.K && k % kGroup8 == 0) p.kept_s[(which * p.M + m) * p.groups + k / kGroup8] = g.s;
  return codes8(v, g);
}

template <typename T>
__device__ __forceinline__ void silu_mul(float (&v)[8], const float (&u)[8]) {
#pragma unroll
  for (int e = 0; e < 8; ++e) v[e] = v[e] * sigmoid<T>(v[e]) * u[e];
}

// 8 values of the row to quantize, any K
template <typename T, bool SILU>
__device__ __forceinline__ void value8(const RowArgs& p, int64_t m, int64_t k, bool keep, float (&v)[8]) {
  load8((const T*)p.x + m * p.ldx, k, p.K, v);
  if constexpr (SILU) {
    float u[8];
    load8((const T*)p.u + m * p.ldu, k, p.K, u);
    if (keep) {
      const uint2 g = keep8(p, 0, m, k, v), h = keep8(p, 1, m, k, u);
      if (k < p.K) {
        store_codes(p.kept_q + m * p.K + k, g, p.K - k);
        store_codes(p.kept_q + (p.M + m) * p.K + k, h, p.K - k);
      }
    }
    silu_mul<T>(v, u);
  }
}

// THREADS threads a row, C chunks of 8 columns a thread (C = 0: any number, the row read twice). Rows of a
// wavefront: 4 a block.
template <typename T, bool SILU, int THREADS, int C>
__global__ __launch_bounds__(THREADS == 64 ? 256 : THREADS) void rows8_kernel(const RowArgs p) {
  constexpr bool WAVE = THREADS == 64;
  const int t = WAVE ? threadIdx.x & 63 : threadIdx.x;
  const int64_t m = p.first + (WAVE ? (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6) : blockIdx.x);
  if (m >= p.M) return;
  const bool keep = SILU && p.kept_q != nullptr;
  float v[C ? C : 1][8];
  uint32_t top = 0;
  auto column = [&](int c) { return (int64_t)(c * THREADS + t) * 8; };
  if constexpr (C != 0) {
    if (p.K % 8 == 0 && p.K > 0) {
      Raw8<T> x[C], u[SILU ? C : 1];
#pragma unroll
      for (int c = 0; c < C; ++c) {
        x[c] = fetch8((const T*)p.x + m * p.ldx, column(c), p.K);
        if constexpr (SILU) u[c] = fetch8((const T*)p.u + m * p.ldu, column(c), p.K);
      }
#pragma unroll
      for (int c = 0; c < C; ++c) widen8(x[c], column(c) < p.K, v[c]);
      if constexpr (SILU) {
        int8_t *kg = p.kept_q + m * p.K, *ku = p.kept_q + (p.M + m) * p.K;
#pragma unroll
        for (int c = 0; c < C; c += 2) {
          const int n = C - c < 2 ? C - c : 2;
          float uv[2][8];
          uint2 g[2], h[2];
#pragma unroll
          for (int d = 0; d < 2; ++d) {
            if (d >= n) continue;
            widen8(u[c + d < C ? c + d : c], column(c + d) < p.K, uv[d]);
            if (keep) {
              g[d] = keep8(p, 0, m, column(c + d), v[c + d < C ? c + d : c]);
              h[d] = keep8(p, 1, m, column(c + d), uv[d]);
            }
          }
          if (keep) {
            if (n == 2 && p.K % 16 == 0) {
              store_two(kg, g[0], g[1], column(c), column(c + 1), p.K, t);
              store_two(ku, h[0], h[1], column(c), column(c + 1), p.K, t);
            } else {
#pragma unroll
              for (int d = 0; d < 2; ++d)
                if (d < n && column(c + d) < p.K) {
                  store_codes(kg + column(c + d), g[d], 8);
                  store_codes(ku + column(c + d), h[d], 8);
                }
            }
          }
#pragma unroll
          for (int d = 0; d < 2; ++d)
            if (d < n) silu_mul<T>(v[c + d < C ? c + d : c], uv[d]);
        }
      }
#pragma unroll
      for (int c = 0; c < C; ++c) top = max(top, max_abs8(v[c]));
    } else {
#pragma unroll
      for (int c = 0; c < C; ++c) {
        value8<T, SILU>(p, m, column(c), keep, v[c]);
        top = max(top, max_abs8(v[c]));
      }
    }
  } else {
    // (whole groups of lanes: keep8 needs them all)
    for (int64_t k0 = 0; k0 < p.K; k0 += THREADS * 8) {
      value8<T, SILU>(p, m, k0 + t * 8, keep, v[0]);
      top = max(top, max_abs8(v[0]));
    }
  }
  top = group_max_bits<64>(top);
  if constexpr (!WAVE) {
    __shared__ uint32_t red[THREADS / 64];
    if ((t & 63) == 0) red[t >> 6] = top;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < THREADS / 64; ++w) top = max(top, red[w]);
  }
  const Scale8 g = scale8(top);
  if (t == 0) p.s[m] = g.s;
  int8_t* q = p.q + m * p.ldq;
  if constexpr (C != 0) {
#pragma unroll
    for (int c = 0; c < C; c += 2) {
      if (c + 1 < C && p.kpad % 16 == 0) {
        store_two(q, codes8(v[c], g), codes8(v[c + 1 < C ? c + 1 : c], g), column(c), column(c + 1), p.kpad, t);
      } else {
#pragma unroll
        for (int d = 0; d < 2; ++d)
          if (c + d < C && column(c + d) < p.kpad)
            store_codes(q + column(c + d), codes8(v[c + d < C ? c + d : c], g), p.kpad - column(c + d));
      }
    }
  } else {
    for (int64_t k = t * 8; k < p.kpad; k += THREADS * 8) {
      value8<T, SILU>(p, m, k, false, v[0]);
      store_codes(q + k, codes8(v[0], g), p.kpad - k);
    }
  }
}

// Rows p.first .. p.first + rows.
template <typename T, bool SILU>
int launch_some_rows(const RowArgs& p, int64_t rows, hipStream_t st, const char* fn) {
  const int64_t chunks = cdiv(p.kpad, 8);
#define MLS_ROWS(TH, C)                                                                                          \
  hipLaunchKernelGGL((rows8_kernel<T, SILU, TH, C>), dim3((unsigned)(TH == 64 ? cdiv(rows, 4) : rows)),          \
                     dim3(TH == 64 ? 256 : TH), 0, st, p)
  // Few rows: as many threads a row as it has chunks, since what a block does takes the longer the more a thread does
  // (one row of 11008 bf16 gates and ups: 512 threads 5.9 us, 1024 4.3). Many: enough rows a CU at a time, blocks of 256.
  // Three chunks where four would leave a quarter of the threads without columns (with the checkpoint's stores: the times at store_two).
  const bool few = p.M <= 512;
  if (chunks <= 64) MLS_ROWS(64, 1);
  else if (chunks <= 128) MLS_ROWS(64, 2);
  else if (chunks <= 256) MLS_ROWS(256, 1);
  else if (chunks <= 512 && few) MLS_ROWS(512, 1);
  else if (chunks <= 512) MLS_ROWS(256, 2);
  else if (chunks <= 1024 && few) MLS_ROWS(1024, 1);
  else if (chunks <= 768) MLS_ROWS(256, 3);
  else if (chunks <= 1024) MLS_ROWS(256, 4);
  else if (chunks <= 2048 && few) MLS_ROWS(1024, 2);
  else if (chunks <= 1536) MLS_ROWS(512, 3);
  else if (chunks <= 2048) MLS_ROWS(512, 4);
  else if (chunks <= 4096) MLS_ROWS(1024, 4);
  else MLS_ROWS(1024, 0);
#undef MLS_ROWS
  return check_launch(fn);
}

template <typename T, bool SILU>
int launch_rows(RowArgs p, hipStream_t st, const char* fn) {
  constexpr int64_t kRows = 1 << 21;  // a launch's most: with 1024 threads each 2^31 threads, and a grid has less than 2^32
  for (; p.M - p.first > kRows; p.first += kRows)
    if (const int rc = launch_some_rows<T, SILU>(p, kRows, st, fn)) return rc;
  return launch_some_rows<T, SILU>(p, p.M - p.first, st, fn);
}

template <bool SILU>
int launch_rows_dt(const RowArgs& p, int dt, hipStream_t st, const char* fn) {
  if (dt == MLS_F32) return launch_rows<float, SILU>(p, st, fn);
  if (dt == MLS_F16) return launch_rows<_Float16, SILU>(p, st, fn);
  return launch_rows<__bf16, SILU>(p, st, fn);
}

__global__ __launch_bounds__(256) void pad_rows_kernel(const PadRows one, const PadRows two, int64_t K, int64_t kpad) {
  const int64_t per = kpad / 16;
  int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const bool second = i >= one.rows * per;
  const PadRows p = second ? two : one;
  if (second) i -= one.rows * per;
  if (i >= p.rows * per) return;
  const int64_t r = i / per, k = (i - r * per) * 16;
  uint4 v = make_uint4(0, 0, 0, 0);
  const uint8_t* s = p.src + r * p.ld + k;
  if (k + 16 <= K) {
    __builtin_memcpy(&v, s, 16);
  } else {
    uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
    for (int e = 0; e < 16; ++e)
      if (k + e < K) w[e / 4] |= (uint32_t)s[e] << (8 * (e % 4));
    v = make_uint4(w[0], w[1], w[2], w[3]);
  }
  *reinterpret_cast<uint4*>(p.dst + r * kpad + k) = v;
}

struct BackArgs {
  const void* dh;
  int64_t lddh;
  const int8_t* q;  // [2][M][H], rows ldq apart, the two qs apart
  int64_t ldq, qs;
  const float* s;   // [2][M][groups]
  int64_t lds, ss;
  void* dg;
  void* du;
  int64_t ldo;
  int64_t M, H, per;  // per: chunks of 8 columns a row
};

template <typename T>
__global__ __launch_bounds__(256) void silu_back_kernel(const BackArgs p) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= p.M * p.per) return;
  const int64_t m = (p.M * p.per) >> 32 ? i / p.per : (uint32_t)i / (uint32_t)p.per, k = (i - m * p.per) * 8;
  const float* s = p.s + m * p.lds + k / kGroup8;
  const int8_t *q0 = p.q + m * p.ldq, *q1 = q0 + p.qs;
  const T* dh = (const T*)p.dh + m * p.lddh;
  float d[8], g[8], u[8];
  if (p.H % 8 == 0) {
    const Raw8<T> raw = fetch8(dh, k, p.H);
    const Raw8<int8_t> c0 = fetch8(q0, k, p.H), c1 = fetch8(q1, k, p.H);
    const float s0 = s[0], s1 = s[p.ss];
    const uint2 w0 = __builtin_bit_cast(uint2, c0), w1 = __builtin_bit_cast(uint2, c1);
    widen8(raw, true, d);
    codes_to_values(w0.x, w0.y, s0, g);
    codes_to_values(w1.x, w1.y, s1, u);
  } else {
    load8(dh, k, p.H, d);
    load_codes8(q0, k, p.H, s[0], g);
    load_codes8(q1, k, p.H, s[p.ss], u);
  }
  float dg[8], du[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const float sig = sigmoid<T>(g[e]), ds = d[e] * sig;
    du[e] = ds * g[e];
    dg[e] = ds * u[e] * (1.0f + g[e] * (1.0f - sig));
  }
  store8((T*)p.dg + m * p.ldo + k, dg, p.H - k);
  store8((T*)p.du + m * p.ldo + k, du, p.H - k);
}

}  // namespace

int launch_quantize_rows(const void* x, int dt, int64_t ldx, int64_t M, int64_t K, int64_t kpad, int8_t* q,
                         int64_t ldq, float* s, hipStream_t st) {
  RowArgs p{};
  p.x = x;
  p.ldx = ldx;
  p.M = M;
  p.K = K;
  p.kpad = kpad;
  p.q = q;
  p.ldq = ldq;
  p.s = s;
  return launch_rows_dt<false>(p, dt, st, "quantize_rows");
}

int launch_pad_rows(const PadRows& one, const PadRows& two, int64_t K, int64_t kpad, hipStream_t st) {
  const int64_t n = cdiv((one.rows + two.rows) * (kpad / 16), 256);
  if (!grid_fits(n, 256)) return fail(MLS_ERR_UNSUPPORTED, "pad rows: %lld x %lld", (long long)(one.rows + two.rows), (long long)K);
  if (n == 0) return MLS_OK;
  hipLaunchKernelGGL(pad_rows_kernel, dim3((unsigned)n), dim3(256), 0, st, one, two, K, kpad);
  return check_launch("pad rows");
}

}  // namespace mls

using namespace mls;

extern "C" int mlsx_quantize_rows(const void* x, int dt, int64_t ldx, int64_t M, int64_t K, int8_t* q, int64_t ldq,
                                  float* s, mls_stream_t stream) {
  const char* fn = "mlsx_quantize_rows";
  if (M < 0 || K < 0) return fail(MLS_ERR_ARG, "%s: negative size", fn);
  if (!is_float_dt(dt)) return fail(MLS_ERR_ARG, "%s: bad dtype %d", fn, dt);
  if (M == 0) return MLS_OK;
  if ((K > 0 && (!x || !q)) || !s) return fail(MLS_ERR_ARG, "%s: null pointer", fn);
  if (ldx < K || ldq < K) return fail(MLS_ERR_ARG, "%s: bad leading dimension", fn);
  return launch_quantize_rows(x, dt, ldx, M, K, K, q, ldq, s, (hipStream_t)stream);
}

extern "C" int mlsx_silu_mul_quantize(const void* gate, int64_t ldg, const void* up, int64_t ldu, int dt, int64_t M,
                                      int64_t H, int8_t* q, int64_t ldq, float* s, int8_t* kept_q, float* kept_s,
                                      mls_stream_t stream) {
  const char* fn = "mlsx_silu_mul_quantize";
  if (M < 0 || H < 0) return fail(MLS_ERR_ARG, "%s: negative size", fn);
  if (!is_float_dt(dt)) return fail(MLS_ERR_ARG, "%s: bad dtype %d", fn, dt);
  if (M == 0) return MLS_OK;
  if ((H > 0 && (!gate || !up || !q)) || !s || (kept_q == nullptr) != (kept_s == nullptr))
    return fail(MLS_ERR_ARG, "%s: null pointer", fn);
  if (ldg < H || ldu < H || ldq < H) return fail(MLS_ERR_ARG, "%s: bad leading dimension", fn);
  RowArgs p{gate, up, ldg, ldu, M, H, H, 0, q, ldq, s, kept_q, kept_s, cdiv(H, kGroup8)};
  return launch_rows_dt<true>(p, dt, (hipStream_t)stream, fn);
}

extern "C" int mlsx_silu_mul_backward(const void* dh, int64_t lddh, int dt, const int8_t* q, int64_t ldq, int64_t q_step,
                                      const float* s, int64_t lds, int64_t s_step, int64_t M, int64_t H, void* dgate,
                                      void* dup, int64_t ldo, mls_stream_t stream) {
  const char* fn = "mlsx_silu_mul_backward";
  if (M < 0 || H < 0) return fail(MLS_ERR_ARG, "%s: negative size", fn);
  if (!is_float_dt(dt)) return fail(MLS_ERR_ARG, "%s: bad dtype %d", fn, dt);
  if (M == 0 || H == 0) return MLS_OK;
  if (!dh || !q || !s || !dgate || !dup) return fail(MLS_ERR_ARG, "%s: null pointer", fn);
  if (lddh < H || ldq < H || lds < cdiv(H, kGroup8) || ldo < H) return fail(MLS_ERR_ARG, "%s: bad leading dimension", fn);
  const BackArgs p{dh, lddh, q, ldq, q_step, s, lds, s_step, dgate, dup, ldo, M, H, cdiv(H, 8)};
  const int64_t n = cdiv(M * p.per, 256);
  if (!grid_fits(n, 256)) return fail(MLS_ERR_UNSUPPORTED, "%s: %lld x %lld", fn, (long long)M, (long long)H);
  const dim3 grid((unsigned)n), block(256);
  if (dt == MLS_F32) hipLaunchKernelGGL(silu_back_kernel<float>, grid, block, 0, (hipStream_t)stream, p);
  else if (dt == MLS_F16) hipLaunchKernelGGL(silu_back_kernel<_Float16>, grid, block, 0, (hipStream_t)stream, p);
  else hipLaunchKernelGGL(silu_back_kernel<__bf16>, grid, block, 0, (hipStream_t)stream, p);
  return check_launch(fn);
}
