// dw[n][k] = sum_m dy[m][n] s[m] q[m][k]: the gradient of a weight whose layer kept its input as 8-bit codes
// with a scale a token.
//
// 16-bit dy: the kept value q s is rounded to dy's type (off by half a step of it, as dy itself is) and the product runs on
// the 16-bit matrix cores with fp32 sums. fp16: the scales may stand for values past 65504 or below 2^-14 (a product of two
// activations is quantized from fp32), so a power of two that brings the largest scale to [2^7, 2^8) is taken out of all and put back
// into the sums: values stay below 2^15, and those of rows with 2^-22 of the largest scale still have all 11 bits. What that rounding
// costs (2100 tokens, 11008 x 4096, bf16): 2.3e-3 of the norm off, where rounding the result alone is 1.7e-3; without it, dy widened
// to fp32 and the result rounded to bf16, 1.7e-3 and 449 us instead of 187 on one box. fp32: dy s, rounded once, becomes three bf16 parts that add up to it
// (8 significant bits each), and each meets the codes, which bf16 holds exactly: three products where two fp32
// operands would take six. Parts of values under 2^-110 lose bits below 2^-133, bf16's smallest.
//
// Both operands are turned first, so that their rows run along the tokens (dw8_turn_kernel; the rows' ends are padded with zeros to
// 64 tokens), then multiplied tile by tile (nt_tile.h). 2100 tokens, 11008 x 4096, bf16: turn 22 us (bytes at a copy's rate 23.6), product 155
// (1.2 PFLOP/s); the library's product of full-width operands 244. fp32, 1000 tokens, 2048 x 1024: 11 and 21, the library's 37.
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
  const float* unit;  // fp16: the power of two that the scales are divided by
  void* dyt;  // [N][Mp]; fp32: bf16 [N][3][Mp]
  void* xt;   // [K][Mp]
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

// unit: the power of two that divides the largest finite scale to [2^7, 2^8). One block.
__global__ __launch_bounds__(1024) void dw8_unit_kernel(const float* s, int M, float* unit) {
  __shared__ uint32_t red[16];
  uint32_t top = 0;
  for (int m = threadIdx.x; m < M; m += 1024) {
    const uint32_t b = abs_bits(s[m]);
    top = max(top, b < 0x7F800000u ? b : 0u);
  }
  top = group_max_bits<64>(top);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = top;
  __syncthreads();
  if (threadIdx.x != 0) return;
  for (int w = 0; w < 16; ++w) top = max(top, red[w]);
  // (an exponent of 1 at least: its reciprocal is a normal number too)
  *unit = __uint_as_float((uint32_t)max((int)(top >> 23) - 7, 1) << 23);
}

// 8 tokens x W columns a lane, turned in registers, 8 x 8 lanes a wavefront: loads take 128 bytes (codes: 64) of each of 8
// rows, stores 128 bytes of 8 of the results' rows. PARTS: of every value (the second and third of what is left).
template <typename T, typename P, int W, int PARTS, bool CODES>
__device__ __forceinline__ void turn(const TurnArgs& p, int C, P* dst) {
  const int c0 = blockIdx.x * 8 * W + (threadIdx.x & 7) * W, m0 = blockIdx.y * 64 + (threadIdx.x >> 3) * 8;
  if (c0 >= C) return;
  float v[8][W];  // [token][column]
  float scale[8];
#pragma unroll
  for (int r = 0; r < 8; ++r) scale[r] = p.s[min(m0 + r, p.M - 1)];
  if constexpr (CODES && __is_same(T, _Float16)) {
    const float inv = 1.0f / *p.unit;
#pragma unroll
    for (int r = 0; r < 8; ++r) scale[r] *= inv;
  }
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
  // 16-bit: codes become values here; fp32: the scale goes to dy
#pragma unroll
  for (int r = 0; r < 8; ++r)
#pragma unroll
    for (int e = 0; e < W; ++e) {
      if constexpr (CODES != (sizeof(T) == 4)) v[r][e] *= scale[r];
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

// blockIdx.z: 0 dy, 1 the kept input
template <typename T>
__global__ __launch_bounds__(64) void dw8_turn_kernel(const TurnArgs p) {
  if constexpr (sizeof(T) == 4) {
    if (blockIdx.z == 0) turn<T, __bf16, 4, 3, false>(p, p.N, (__bf16*)p.dyt);
    else turn<T, __bf16, 8, 1, true>(p, p.K, (__bf16*)p.xt);
  } else {
    if (blockIdx.z == 0) turn<T, T, 8, 1, false>(p, p.N, (T*)p.dyt);
    else turn<T, T, 8, 1, true>(p, p.K, (T*)p.xt);
  }
}

struct Dw8Args {
  NtOperands o;
  void* c;  // direct: OT [N][ldc]; partial: fp32 [splits][N][K]
  int64_t ldc;
  int m_tiles, n_tiles, splits;
  const float* unit;  // fp16: as the scales were divided by it
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
  if constexpr (!PARTIAL && __is_same(P, _Float16)) {
    const float unit = *p.unit;
#pragma unroll
    for (int i = 0; i < G::TN; ++i)
#pragma unroll
      for (int j = 0; j < G::TM; ++j) acc[i][j] *= unit;
  }
  const bool wide = (p.ldc * sizeof(CT)) % 16 == 0 && ((uintptr_t)p.c & 15) == 0;
  const int M = p.o.M, N = p.o.N, m0 = G::row(mt * G::BM, wave, lane), n0 = G::column(nt * G::BN, wave, lane);
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
                                                       int64_t ldc, int N, int K, const float* __restrict__ unit) {
  const int k = (blockIdx.x * 256 + threadIdx.x) * 4, n = blockIdx.y;
  if (k >= K) return;
  const float* src = part + n * ldp + k;
  float4 v = *reinterpret_cast<const float4*>(src);
  for (int i = 1; i < splits; ++i) {
    const float4 q = *reinterpret_cast<const float4*>(src + i * N * ldp);
    v.x += q.x; v.y += q.y; v.z += q.z; v.w += q.w;
  }
  const float u = __is_same(P, _Float16) ? *unit : 1.0f, o[4] = {v.x * u, v.y * u, v.z * u, v.w * u};
#pragma unroll
  for (int e = 0; e < 4; ++e)
    if (k + e < K) c[n * ldc + k + e] = from_f32<CT>(o[e]);
}

struct DwPlan {
  int64_t Mp, xt_at, unit_at, part_at, ldp, bytes;
  int form, splits;
};

int64_t up256(int64_t v) { return (v + 255) / 256 * 256; }

DwPlan make_plan(int dt, int64_t M, int64_t N, int64_t K) {
  DwPlan p{};
  const int parts = dt == MLS_F32 ? 3 : 1;
  p.Mp = cdiv(M, 64) * 64;
  p.xt_at = up256(N * parts * p.Mp * 2);
  p.unit_at = p.xt_at + up256(K * p.Mp * 2);
  p.part_at = p.unit_at + 256;
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
        if (const int rc = launch_dw8<P, OT, G, true>(b, st)) return rc;
        hipLaunchKernelGGL((dw8_join_kernel<P, OT>), dim3((unsigned)cdiv(a.o.N, 1024), (unsigned)a.o.M), dim3(256), 0, st, (const float*)part,
                           a.splits, ldp, (OT*)a.c, a.ldc, a.o.M, a.o.N, a.unit);
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
  float* unit = (float*)(ws + p.unit_at);
  if constexpr (__is_same(T, _Float16)) {
    hipLaunchKernelGGL(dw8_unit_kernel, dim3(1), dim3(1024), 0, st, t.s, t.M, unit);
    if (const int rc = check_launch(fn)) return rc;
  }
  hipLaunchKernelGGL(dw8_turn_kernel<T>, dim3((unsigned)std::max(cdiv(t.N, sizeof(T) == 4 ? 32 : 64), cdiv(t.K, 64)), (unsigned)(p.Mp / 64), 2), dim3(64), 0, st, t);
  if (const int rc = check_launch(fn)) return rc;
  const int parts = sizeof(T) == 4 ? 3 : 1, ld = (int)p.Mp * 2;
  using P = std::conditional_t<sizeof(T) == 4, __bf16, T>;
  const Dw8Args a{{ws, ws + p.xt_at, parts * ld, ld, t.N, t.K, parts * ld, parts}, dw, lddw, 0, 0, p.splits, unit};
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
  const TurnArgs t{dy, lddy, q, ldq, s, (int)M, (int)N, (int)K, (int)p.Mp, (const float*)(w + p.unit_at), w, w + p.xt_at};
  if (dt == MLS_F32) return run<float>(t, dw, dw_dt, lddw, p, w, st);
  if (dt == MLS_F16) return run<_Float16>(t, dw, dw_dt, lddw, p, w, st);
  return run<__bf16>(t, dw, dw_dt, lddw, p, w, st);
}

extern "C" int mlsx_dw_int8(const void* dy, int dt, int64_t lddy, const int8_t* q, int64_t ldq, const float* s, void* dw,
                            int64_t lddw, int64_t M, int64_t N, int64_t K, void* ws, int64_t ws_bytes, mls_stream_t stream) {
  return mlsx_dw_int8_to(dy, dt, lddy, q, ldq, s, dw, dt, lddw, M, N, K, ws, ws_bytes, stream);
}
