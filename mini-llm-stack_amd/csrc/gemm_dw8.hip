// dw[n][k] = sum_m dy[m][n] s[m] q[m][k]: the gradient of a weight whose layer kept its input as 8-bit codes
// with a scale a token.
//
// 16-bit dy: on the fp16 matrix cores, with fp32 sums. A token's scale is f 2^e, f in [1/2, 1): f goes to the codes, rounded to fp16's 11
// bits (which a code and a scale need 32 of), and 2^e to dy, whose bits stay as they are. So that dy 2^e fits fp16's range, it is held in units of a power of
// two a column, found first: the column's largest at [2^14, 2^15). Numbers of 2^-32 of that (fp16: 2^-28) are still exact, smaller ones
// are on a grid of 2^-39. The power is put back into the sums. (2100 tokens, 11008 x 4096, bf16: 1.67e-3 of the norm off, as the rounding of
// the result alone, 190 us; with the kept value rounded to bf16 instead, which needs no pass over dy's columns, 2.36e-3 and 175; with three parts as fp32, 450.)
// fp32: dy s, rounded once, becomes three bf16 parts that add up to it
// (8 significant bits each), and each meets the codes, which bf16 holds exactly: three products where two fp32
// operands would take six. Parts of values under 2^-110 lose bits below 2^-133, bf16's smallest.
//
// Both operands are turned first, so that their rows run along the tokens (the rows' ends are padded with zeros to
// 64 tokens), then multiplied tile by tile (nt_tile.h). The same call: exponents and the codes' turn 15 us, dy's 19 (92 MB, 4.9 TB/s), product 160
// (1.2 PFLOP/s); the library's product of full-width operands 244. fp32, 1000 tokens, 2048 x 1024: 11 and 22, the library's 37.
#include <algorithm>
#include <type_traits>

#include "act8.h"
#include "mfma16.h"
#include "nt_tile.h"

namespace mls {

namespace {

template <typename T>
struct Op16 {
  using Acc = f32x4;
  __device__ static __forceinline__ f32x4 mma(const i32x4& a, const i32x4& b, const f32x4& c) {
    return Mfma16<T>::mma(__builtin_bit_cast(uint4, a), __builtin_bit_cast(uint4, b), c);
  }
};

struct TurnArgs {
  const void* dy;
  int64_t lddy;
  const int8_t* q;
  int64_t ldq;
  const float* s;
  int M, N, K, Mp;
  void* dyt;  // fp16 [N][Mp]; fp32: bf16 [N][3][Mp]
  void* xt;   // [K][Mp]
  // 16-bit dy: columns' exponents, rows of N8 (N rounded up to 8): of each of `chunks` parts of the tokens, and of all
  int16_t *some, *exps;
  int chunks, N8;
};

// n <= W consecutive values of a row, zeros past them
template <int W, typename T>
__device__ __forceinline__ void load_some(const T* src, int64_t n, float (&v)[W]) {
  T raw[W];
  if (n >= W) {
    __builtin_memcpy(raw, src, sizeof(raw));
#pragma unroll
    for (int e = 0; e < W; ++e) v[e] = to_f32(raw[e]);
  } else {
#pragma unroll
    for (int e = 0; e < W; ++e) v[e] = e < n ? to_f32(src[e]) : 0.0f;
  }
}

typedef int16_t i16x8 __attribute__((ext_vector_type(8)));

// Over the 8 lanes of a wavefront that hold the same columns.
__device__ __forceinline__ i16x8 max_of_tokens(i16x8 v) {
  uint4 w = __builtin_bit_cast(uint4, v);
#pragma unroll
  for (int d = 8; d < 64; d *= 2) {
    const uint4 o = make_uint4(__shfl_xor(w.x, d, 64), __shfl_xor(w.y, d, 64), __shfl_xor(w.z, d, 64), __shfl_xor(w.w, d, 64));
    v = __builtin_elementwise_max(v, __builtin_bit_cast(i16x8, o));
    w = __builtin_bit_cast(uint4, v);
  }
  return v;
}

constexpr int16_t kNoExponent = -16384;  // of a column of zeros

// The largest e of |dy 2^(a scale's exponent)| < 2^e over a part of the tokens, of 64 columns a wavefront, 8 a lane. Zeros and
// what is no finite number do not count. A number's bits and the scale's exponent in the place of its own add up: the largest of
// these sums has the exponent that is looked for, over a bias.
template <typename T>
__device__ __forceinline__ void column_exponents(const TurnArgs& p) {
  constexpr int SHIFT = __is_same(T, _Float16) ? 10 : 7, ALL = 0x7FFF >> SHIFT, BIAS = ALL / 2 - 1;
  constexpr int NONE = (kNoExponent + BIAS) * (1 << SHIFT);
  const int c0 = blockIdx.x * 64 + (threadIdx.x & 7) * 8, r = threadIdx.x >> 3;
  if ((int)blockIdx.y >= p.chunks || (int)blockIdx.x * 64 >= p.N) return;
  const int lo = (int)((int64_t)p.M * blockIdx.y / p.chunks), hi = (int)((int64_t)p.M * (blockIdx.y + 1) / p.chunks);
  const bool whole = c0 + 8 <= p.N;
  int top[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) top[e] = NONE;
  for (int m0 = lo + r; m0 < hi + r; m0 += 64) {
    uint4 raw[8];
    float s[8];
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      const int64_t m = min(m0 + 8 * u, hi - 1);  // (some twice: a maximum)
      const uint16_t* src = (const uint16_t*)p.dy + m * p.lddy + c0;
      s[u] = p.s[m];
      if (whole) {
        __builtin_memcpy(&raw[u], src, 16);
      } else {
        uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (c0 + e < p.N) w[e / 2] |= (uint32_t)src[e] << (16 * (e % 2));
        raw[u] = make_uint4(w[0], w[1], w[2], w[3]);
      }
    }
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      const uint32_t w[4] = {raw[u].x, raw[u].y, raw[u].z, raw[u].w};
      const int x = __builtin_amdgcn_frexp_expf(s[u]) * (1 << SHIFT);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const uint32_t b = (w[e / 2] >> (16 * (e % 2))) & 0x7FFFu;
        top[e] = max(top[e], b - 1u < (uint32_t)(ALL << SHIFT) - 1u ? (int)b + x : NONE);
      }
    }
  }
  i16x8 all;
#pragma unroll
  for (int e = 0; e < 8; ++e) all[e] = (int16_t)((top[e] >> SHIFT) - BIAS);
  all = max_of_tokens(all);
  if (r == 0 && c0 < p.N) *reinterpret_cast<i16x8*>(p.some + (int64_t)blockIdx.y * p.N8 + c0) = all;
}

// 8 tokens x W columns a lane, turned in registers, 8 x 8 lanes a wavefront: loads take 128 bytes (codes: 64) of each of 8
// rows, stores 128 bytes of 8 of the results' rows. PARTS: of every value (the second and third of what is left).
template <typename T, typename P, int W, int PARTS, bool CODES>
__device__ __forceinline__ void turn(const TurnArgs& p, int C, P* dst) {
  const int c0 = blockIdx.x * 8 * W + (threadIdx.x & 7) * W, m0 = blockIdx.y * 64 + (threadIdx.x >> 3) * 8;
  i16x8 unit;  // 16-bit dy: the columns' powers of two
  if constexpr (sizeof(T) == 2 && !CODES) {
    unit = kNoExponent;
    if (c0 < C)
      for (int i = threadIdx.x >> 3; i < p.chunks; i += 8)
        unit = __builtin_elementwise_max(unit, *reinterpret_cast<const i16x8*>(p.some + (int64_t)i * p.N8 + c0));
    unit = max_of_tokens(unit) - (int16_t)15;
    if (c0 < C && m0 == 0) *reinterpret_cast<i16x8*>(p.exps + c0) = unit;
  }
  if (c0 >= C) return;
  float v[8][W];  // [token][column]
  float scale[8];
#pragma unroll
  for (int r = 0; r < 8; ++r) scale[r] = p.s[min(m0 + r, p.M - 1)];
  if ((int)(blockIdx.x + 1) * 8 * W <= C) {
    // without branches, so that all rows are on their way at once
    using Raw = std::conditional_t<CODES, int8_t, T>;
    const Raw* src = CODES ? (const Raw*)p.q : (const Raw*)p.dy;
    const int64_t ld = CODES ? p.ldq : p.lddy;
    Raw raw[8][W];
#pragma unroll
    for (int r = 0; r < 8; ++r) __builtin_memcpy(raw[r], src + min(m0 + r, p.M - 1) * ld + c0, sizeof(raw[r]));
#pragma unroll
    for (int r = 0; r < 8; ++r)
#pragma unroll
      for (int e = 0; e < W; ++e) {
        if constexpr (CODES) v[r][e] = (float)raw[r][e];
        else v[r][e] = to_f32(raw[r][e]);
      }
  } else {
#pragma unroll
    for (int r = 0; r < 8; ++r) {
      const int64_t m = min(m0 + r, p.M - 1);
      if constexpr (CODES) load_codes8(p.q + m * p.ldq, c0, C, 1.0f, v[r]);
      else load_some<W>((const T*)p.dy + m * p.lddy + c0, C - c0, v[r]);
    }
  }
#pragma unroll
  for (int r = 0; r < 8; ++r)
#pragma unroll
    for (int e = 0; e < W; ++e) {
      if constexpr (sizeof(T) == 2 && CODES) v[r][e] *= __builtin_amdgcn_frexp_mantf(scale[r]);
      if constexpr (sizeof(T) == 2 && !CODES) v[r][e] = __builtin_amdgcn_ldexpf(v[r][e], __builtin_amdgcn_frexp_expf(scale[r]) - unit[e]);
      if constexpr (sizeof(T) == 4 && !CODES) v[r][e] *= scale[r];
      if (m0 + r >= p.M) v[r][e] = 0.0f;
    }
#pragma unroll
  for (int c = 0; c < W; ++c) {
    if (c0 + c >= C) continue;
#pragma unroll
    for (int t = 0; t < PARTS; ++t) {
      P o[8];
#pragma unroll
      for (int r = 0; r < 8; ++r) {
        float part = v[r][c];
        if (t + 1 < PARTS) split_f32(v[r][c], part, v[r][c]);
        o[r] = (P)part;
      }
      __builtin_memcpy(__builtin_assume_aligned(dst + ((int64_t)(c0 + c) * PARTS + t) * p.Mp + m0, 16), o, 16);
    }
  }
}

// fp32. blockIdx.z: 0 dy, 1 the kept input
__global__ __launch_bounds__(64) void dw8_turn_kernel(const TurnArgs p) {
  if (blockIdx.z == 0) turn<float, __bf16, 4, 3, false>(p, p.N, (__bf16*)p.dyt);
  else turn<float, __bf16, 8, 1, true>(p, p.K, (__bf16*)p.xt);
}

// 16-bit: the columns' exponents beside the kept input's turn, then dy's.
template <typename T>
__global__ __launch_bounds__(64) void dw8_prepare_kernel(const TurnArgs p) {
  if (blockIdx.z == 0) column_exponents<T>(p);
  else turn<T, _Float16, 8, 1, true>(p, p.K, (_Float16*)p.xt);
}
template <typename T>
__global__ __launch_bounds__(64) void dw8_turn_dy_kernel(const TurnArgs p) {
  turn<T, _Float16, 8, 1, false>(p, p.N, (_Float16*)p.dyt);
}

// ---------------------------------------------------------------- a bias's gradient: dy's sums over tokens
//
// Bound by reading dy: bf16, 4096 x 11008 19.8 us a call (4.6 TB/s), 2048 x 4096 11.1, 64 x 4096 8.6 (its host work). The weight gradient's kernels with an input of
// ones, which this was, took 68, 30 and 26.

struct SumArgs {
  const void* dy;
  int64_t lddy;
  int M, N, N8, chunks;
  float* some;  // [chunks][N8]
  void* out;
  int out_dt;
};

__device__ __forceinline__ void store_sum(const SumArgs& p, int n, float v) {
  if (p.out_dt == MLS_F32) ((float*)p.out)[n] = v;
  else if (p.out_dt == MLS_F16) ((_Float16*)p.out)[n] = from_f32<_Float16>(v);
  else ((__bf16*)p.out)[n] = from_f32<__bf16>(v);
}

// A wavefront: 64 columns of a part of the tokens, 8 a lane, 8 tokens at a time, in an order that sizes alone decide.
template <typename T>
__global__ __launch_bounds__(64) void column_sums_kernel(const SumArgs p) {
  const int c0 = blockIdx.x * 64 + (threadIdx.x & 7) * 8, r = threadIdx.x >> 3;
  const int lo = (int)((int64_t)p.M * blockIdx.y / p.chunks), hi = (int)((int64_t)p.M * (blockIdx.y + 1) / p.chunks);
  float sum[8] = {0, 0, 0, 0, 0, 0, 0, 0};
  for (int m0 = lo + r; m0 < hi + r; m0 += 64) {
    float v[8][8];
    if (c0 + 8 <= p.N) {
      Raw8<T> raw[8];
#pragma unroll
      for (int u = 0; u < 8; ++u) __builtin_memcpy(&raw[u], (const T*)p.dy + (int64_t)min(m0 + 8 * u, hi - 1) * p.lddy + c0, sizeof(raw[u]));
#pragma unroll
      for (int u = 0; u < 8; ++u) widen8(raw[u], m0 + 8 * u < hi, v[u]);
    } else {
#pragma unroll
      for (int u = 0; u < 8; ++u)
        load8((const T*)p.dy + (int64_t)min(m0 + 8 * u, hi - 1) * p.lddy, c0, m0 + 8 * u < hi ? p.N : 0, v[u]);
    }
#pragma unroll
    for (int u = 0; u < 8; ++u)
#pragma unroll
      for (int e = 0; e < 8; ++e) sum[e] += v[u][e];
  }
#pragma unroll
  for (int e = 0; e < 8; ++e)
#pragma unroll
    for (int d = 8; d < 64; d *= 2) sum[e] += __shfl_xor(sum[e], d, 64);
  if (r != 0) return;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    if (c0 + e >= p.N) continue;
    if (p.chunks == 1) store_sum(p, c0 + e, sum[e]);
    else p.some[(int64_t)blockIdx.y * p.N8 + c0 + e] = sum[e];
  }
}

__global__ __launch_bounds__(64) void join_sums_kernel(const SumArgs p) {
  const int n = blockIdx.x * 64 + threadIdx.x;
  if (n >= p.N) return;
  float v = 0;
#pragma unroll 8
  for (int i = 0; i < p.chunks; ++i) v += p.some[(int64_t)i * p.N8 + n];
  store_sum(p, n, v);
}

// Parts of 64 tokens, or what makes 128 of them.
int sum_chunks(int64_t M) { return (int)std::min<int64_t>(cdiv(M, 64), 128); }

// ---------------------------------------------------------------- the product

struct Dw8Args {
  NtOperands o;
  void* c;  // direct: OT [N][ldc]; partial: fp32 [splits][N][K]
  int64_t ldc;
  int m_tiles, n_tiles, splits;
  const int16_t* exps;  // fp16 operands: the powers of two that a's rows are in units of
};

// P: the operands' type, OT: the gradient's, G: a form of tile
template <typename P, typename OT, class G, bool PARTIAL>
__global__ __launch_bounds__(G::THREADS) void dw8_kernel(const Dw8Args p) {
  extern __shared__ __align__(16) uint8_t lds[];
  int sp, mt, nt;
  nt_place(p.m_tiles, p.n_tiles, sp, mt, nt);
  const int units = (p.o.K + 127) / 128;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  f32x4 acc[G::TN][G::TM];
  if (!G::run(p.o, lds, mt * G::BM, nt * G::BN, (int)((int64_t)units * sp / p.splits), (int)((int64_t)units * (sp + 1) / p.splits), wave,
              lane, acc))
    return;
  using CT = std::conditional_t<PARTIAL, float, OT>;
  CT* c = (CT*)p.c + (PARTIAL ? (int64_t)sp * p.o.M * p.ldc : 0);
  const bool wide = (p.ldc * sizeof(CT)) % 16 == 0 && ((uintptr_t)p.c & 15) == 0;
  const int M = p.o.M, N = p.o.N, m0 = G::row(mt * G::BM, wave, lane), n0 = G::column(nt * G::BN, wave, lane);
  if constexpr (!PARTIAL && __is_same(P, _Float16)) {
    int x[G::TM];
#pragma unroll
    for (int j = 0; j < G::TM; ++j) x[j] = p.exps[min(m0 + 16 * j, M - 1)];
#pragma unroll
    for (int i = 0; i < G::TN; ++i)
#pragma unroll
      for (int j = 0; j < G::TM; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[i][j][e] = __builtin_amdgcn_ldexpf(acc[i][j][e], x[j]);
  }
  if constexpr (sizeof(CT) == 2) {
    const int lk = lane >> 4, nt0 = n0 - 4 * lk;
#pragma unroll
    for (int i = 0; i < G::TN; i += 2)
#pragma unroll
      for (int j = 0; j < G::TM; ++j) {
        uint2 o[2];
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          const f32x4 v = acc[i + t][j];
          o[t] = make_uint2(pack2_bits(from_f32<CT>(v[0]), from_f32<CT>(v[1])), pack2_bits(from_f32<CT>(v[2]), from_f32<CT>(v[3])));
        }
        const int m = m0 + 16 * j;
        nt_store_pair((uint16_t*)c + (int64_t)m * p.ldc + nt0 + 16 * i, nt0 + 16 * i, N, o[0], o[1], lk, m < M, wide);
      }
  } else {
#pragma unroll
    for (int i = 0; i < G::TN; ++i)
#pragma unroll
      for (int j = 0; j < G::TM; ++j) {
        const int m = m0 + 16 * j, n = n0 + 16 * i;
        if (m >= M || n >= N) continue;
        const f32x4 v = acc[i][j];
        CT* dst = c + m * p.ldc + n;
        if (n + 3 < N && wide) {
          store4<CT>(dst, v[0], v[1], v[2], v[3]);
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (n + e < N) dst[e] = from_f32<CT>(v[e]);
        }
      }
  }
}

// Adds the ranges' sums in their order: 4 columns a thread; part [splits][N][ldp], ldp a multiple of 4.
template <typename P, typename CT>
__global__ __launch_bounds__(256) void dw8_join_kernel(const float* __restrict__ part, int splits, int64_t ldp, CT* __restrict__ c,
                                                       int64_t ldc, int N, int K, const int16_t* __restrict__ exps) {
  const int k = (blockIdx.x * 256 + threadIdx.x) * 4, n = blockIdx.y;
  if (k >= K) return;
  const float* src = part + n * ldp + k;
  float4 v = *reinterpret_cast<const float4*>(src);
  for (int i = 1; i < splits; ++i) {
    const float4 q = *reinterpret_cast<const float4*>(src + i * N * ldp);
    v.x += q.x; v.y += q.y; v.z += q.z; v.w += q.w;
  }
  const int x = __is_same(P, _Float16) ? exps[n] : 0;
  const float o[4] = {__builtin_amdgcn_ldexpf(v.x, x), __builtin_amdgcn_ldexpf(v.y, x), __builtin_amdgcn_ldexpf(v.z, x), __builtin_amdgcn_ldexpf(v.w, x)};
#pragma unroll
  for (int e = 0; e < 4; ++e)
    if (k + e < K) c[n * ldc + k + e] = from_f32<CT>(o[e]);
}

struct DwPlan {
  int64_t Mp, xt_at, some_at, exps_at, part_at, ldp, N8, bytes;
  int form, splits, chunks;
};

int64_t up256(int64_t v) { return (v + 255) / 256 * 256; }

DwPlan make_plan(int dt, int64_t M, int64_t N, int64_t K) {
  DwPlan p{};
  const int parts = dt == MLS_F32 ? 3 : 1;
  p.Mp = cdiv(M, 64) * 64;
  p.xt_at = up256(N * parts * p.Mp * 2);
  p.some_at = p.xt_at + up256(K * p.Mp * 2);
  p.exps_at = p.part_at = p.some_at;
  if (dt != MLS_F32) {
    // parts of the tokens, a wavefront each and 64 columns: 64 tokens, or what makes 64 parts, which cost a lane of the turn 8 loads
    p.N8 = cdiv(N, 8) * 8;
    p.chunks = (int)std::min<int64_t>(cdiv(M, 64), 64);
    p.exps_at = p.some_at + up256(p.chunks * p.N8 * 2);
    p.part_at = p.exps_at + up256(p.N8 * 2);
  }
  p.bytes = p.part_at;
  nt_choose(N, K, parts * p.Mp * 2, p.form, p.splits);
  if (p.splits > 1) {
    p.ldp = cdiv(K, 4) * 4;
    p.bytes += up256(p.splits * N * p.ldp * 4);
  }
  return p;
}

template <typename P, typename OT, class G, bool PARTIAL>
int launch_dw8(Dw8Args a, hipStream_t st) {
  const char* fn = "mlsx_dw_int8";
  a.m_tiles = (int)cdiv(a.o.M, G::BM);
  a.n_tiles = (int)cdiv(a.o.N, G::BN);
  const int64_t blocks = (int64_t)a.m_tiles * a.n_tiles * a.splits;
  if (!grid_fits(blocks, G::THREADS)) return fail(MLS_ERR_UNSUPPORTED, "%s: %d x %d", fn, a.o.M, a.o.N);
  auto kern = dw8_kernel<P, OT, G, PARTIAL>;
  // (a call a launch: the limit is the function's on the current device)
  if (hipFuncSetAttribute((const void*)kern, hipFuncAttributeMaxDynamicSharedMemorySize, G::LDS) != hipSuccess)
    return fail(MLS_ERR_HIP, "%s: cannot reserve %d bytes of LDS", fn, G::LDS);
  hipLaunchKernelGGL(kern, dim3((unsigned)blocks), dim3(G::THREADS), G::LDS, st, a);
  return check_launch(fn);
}

// The product of turned operands.
template <typename P, typename OT>
int run_product(Dw8Args a, int64_t ldp, int form, void* part, hipStream_t st) {
  return nt_form<Op16<P>>(form, [&](auto f) {
    using G = typename decltype(f)::type;
    if constexpr (G::RANGES) {
      if (a.splits > 1) {
        Dw8Args b = a;
        b.c = part;
        b.ldc = ldp;
        if (const int rc = launch_dw8<P, float, G, true>(b, st)) return rc;
        hipLaunchKernelGGL((dw8_join_kernel<P, OT>), dim3((unsigned)cdiv(a.o.N, 1024), (unsigned)a.o.M), dim3(256), 0, st, (const float*)part,
                           a.splits, ldp, (OT*)a.c, a.ldc, a.o.M, a.o.N, a.exps);
        return check_launch("mlsx_dw_int8");
      }
    }
    return launch_dw8<P, OT, G, false>(a, st);
  });
}

// T: dy's type
template <typename T>
int run(const TurnArgs& t, void* dw, int dw_dt, int64_t lddw, const DwPlan& p, uint8_t* ws, hipStream_t st) {
  const char* fn = "mlsx_dw_int8";
  const unsigned across = (unsigned)std::max(cdiv(t.N, sizeof(T) == 4 ? 32 : 64), cdiv(t.K, 64)), down = (unsigned)(p.Mp / 64);
  if constexpr (sizeof(T) == 4) {
    hipLaunchKernelGGL(dw8_turn_kernel, dim3(across, down, 2), dim3(64), 0, st, t);
  } else {
    hipLaunchKernelGGL(dw8_prepare_kernel<T>, dim3(across, down, 2), dim3(64), 0, st, t);
    if (const int rc = check_launch(fn)) return rc;
    hipLaunchKernelGGL(dw8_turn_dy_kernel<T>, dim3((unsigned)cdiv(t.N, 64), down), dim3(64), 0, st, t);
  }
  if (const int rc = check_launch(fn)) return rc;
  const int parts = sizeof(T) == 4 ? 3 : 1, ld = (int)p.Mp * 2;
  using P = std::conditional_t<sizeof(T) == 4, __bf16, _Float16>;
  const Dw8Args a{{ws, ws + p.xt_at, parts * ld, ld, t.N, t.K, parts * ld, parts}, dw, lddw, 0, 0, p.splits, t.exps};
  void* part = ws + p.part_at;
  if (dw_dt == MLS_F32) return run_product<P, float>(a, p.ldp, p.form, part, st);
  if (dw_dt == MLS_F16) return run_product<P, _Float16>(a, p.ldp, p.form, part, st);
  return run_product<P, __bf16>(a, p.ldp, p.form, part, st);
}

}  // namespace

}  // namespace mls

using namespace mls;

extern "C" int64_t mlsx_dw_int8_workspace(int dt, int64_t M, int64_t N, int64_t K) {
  if (M < 1 || N < 1 || K < 1 || M > (1 << 20) || N > (1 << 22) || K > (1 << 22)) return 0;
  return make_plan(dt, M, N, K).bytes;
}

extern "C" int64_t mlsx_bias_grad_workspace(int64_t M, int64_t N) {
  if (M < 1 || N < 1 || sum_chunks(M) == 1) return 0;
  return (int64_t)sum_chunks(M) * (cdiv(N, 8) * 8) * 4;
}

extern "C" int mlsx_bias_grad(const void* dy, int dt, int64_t lddy, void* db, int db_dt, int64_t M, int64_t N, void* ws, int64_t ws_bytes,
                              mls_stream_t stream) {
  const char* fn = "mlsx_bias_grad";
  if (M < 1 || N < 0) return fail(MLS_ERR_ARG, "%s: bad size", fn);
  if (!is_float_dt(dt) || !is_float_dt(db_dt)) return fail(MLS_ERR_ARG, "%s: bad dtype %d, %d", fn, dt, db_dt);
  if (N == 0) return MLS_OK;
  if (M > (1 << 30) || N > (1 << 26)) return fail(MLS_ERR_UNSUPPORTED, "%s: M=%lld N=%lld", fn, (long long)M, (long long)N);
  const int64_t need = mlsx_bias_grad_workspace(M, N);
  if (!dy || !db || (need && !ws)) return fail(MLS_ERR_ARG, "%s: null pointer", fn);
  if (lddy < N) return fail(MLS_ERR_ARG, "%s: bad leading dimension", fn);
  if (ws_bytes < need || !aligned(ws, 16)) return fail(MLS_ERR_ARG, "%s: workspace too small or misaligned", fn);
  const SumArgs p{dy, lddy, (int)M, (int)N, (int)(cdiv(N, 8) * 8), sum_chunks(M), (float*)ws, db, db_dt};
  const dim3 grid((unsigned)cdiv(N, 64), (unsigned)p.chunks);
  const hipStream_t st = (hipStream_t)stream;
  if (dt == MLS_F32) hipLaunchKernelGGL(column_sums_kernel<float>, grid, dim3(64), 0, st, p);
  else if (dt == MLS_F16) hipLaunchKernelGGL(column_sums_kernel<_Float16>, grid, dim3(64), 0, st, p);
  else hipLaunchKernelGGL(column_sums_kernel<__bf16>, grid, dim3(64), 0, st, p);
  if (const int rc = check_launch(fn)) return rc;
  if (p.chunks == 1) return MLS_OK;
  hipLaunchKernelGGL(join_sums_kernel, dim3((unsigned)cdiv(N, 64)), dim3(64), 0, st, p);
  return check_launch(fn);
}

extern "C" int mlsx_dw_int8_form(int dt, int64_t M, int64_t N, int64_t K) {
  if (!is_float_dt(dt) || mlsx_dw_int8_workspace(dt, M, N, K) == 0) return -1;
  const DwPlan p = make_plan(dt, M, N, K);
  return 16 * (p.form + 1) + p.splits;
}

extern "C" int mlsx_dw_int8_to(const void* dy, int dt, int64_t lddy, const int8_t* q, int64_t ldq, const float* s, void* dw, int dw_dt,
                               int64_t lddw, int64_t M, int64_t N, int64_t K, void* ws, int64_t ws_bytes, mls_stream_t stream) {
  const char* fn = "mlsx_dw_int8";
  if (M < 1 || N < 0 || K < 0) return fail(MLS_ERR_ARG, "%s: bad size", fn);
  if (!is_float_dt(dt) || !is_float_dt(dw_dt)) return fail(MLS_ERR_ARG, "%s: bad dtype %d, %d", fn, dt, dw_dt);
  if (N == 0 || K == 0) return MLS_OK;
  const int64_t need = mlsx_dw_int8_workspace(dt, M, N, K);
  if (need == 0) return fail(MLS_ERR_UNSUPPORTED, "%s: M=%lld N=%lld K=%lld", fn, (long long)M, (long long)N, (long long)K);
  if (!dy || !q || !s || !dw || !ws) return fail(MLS_ERR_ARG, "%s: null pointer", fn);
  if (lddy < N || ldq < K || lddw < K) return fail(MLS_ERR_ARG, "%s: bad leading dimension", fn);
  if (ws_bytes < need || !aligned(ws, 16)) return fail(MLS_ERR_ARG, "%s: workspace too small or misaligned", fn);
  const DwPlan p = make_plan(dt, M, N, K);
  const hipStream_t st = (hipStream_t)stream;
  uint8_t* w = (uint8_t*)ws;
  const TurnArgs t{dy, lddy, q, ldq, s, (int)M, (int)N, (int)K, (int)p.Mp, w, w + p.xt_at, (int16_t*)(w + p.some_at), (int16_t*)(w + p.exps_at),
                   p.chunks, (int)p.N8};
  if (dt == MLS_F32) return run<float>(t, dw, dw_dt, lddw, p, w, st);
  if (dt == MLS_F16) return run<_Float16>(t, dw, dw_dt, lddw, p, w, st);
  return run<__bf16>(t, dw, dw_dt, lddw, p, w, st);
}

extern "C" int mlsx_dw_int8(const void* dy, int dt, int64_t lddy, const int8_t* q, int64_t ldq, const float* s, void* dw,
                            int64_t lddw, int64_t M, int64_t N, int64_t K, void* ws, int64_t ws_bytes, mls_stream_t stream) {
  return mlsx_dw_int8_to(dy, dt, lddy, q, ldq, s, dw, dt, lddw, M, N, K, ws, ws_bytes, stream);
}
