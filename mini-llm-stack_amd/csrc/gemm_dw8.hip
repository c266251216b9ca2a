// dw[n][k] = sum_m dy[m][n] s[m] q[m][k]: the gradient of a weight whose layer kept its input as 8-bit codes
// with a scale a token.
//
// 16-bit dy: the kept value q s is rounded to dy's type (off by half a step of it, as dy itself is) and the product runs on
// the 16-bit matrix cores with fp32 sums. Both operands are turned first, so that their rows run along the
// tokens (dw8_turn_kernel), then multiplied tile by tile (nt_tile.h).
#include <algorithm>

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
  void* dyt;  // [N][Mp]
  void* xt;   // [K][Mp]
};

// 64 tokens x 64 columns through LDS. blockIdx.z: 0 dy, 1 the kept input. Tokens past M become zeros.
template <typename T>
__global__ __launch_bounds__(256) void dw8_turn_kernel(const TurnArgs p) {
  __shared__ T tile[64][72];
  const bool second = blockIdx.z != 0;
  const int C = second ? p.K : p.N, c0 = blockIdx.x * 64, m0 = blockIdx.y * 64, tid = threadIdx.x;
  if (c0 >= C) return;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int r = i * 32 + tid / 8, c = (tid % 8) * 8, m = m0 + r;
    float v[8] = {0, 0, 0, 0, 0, 0, 0, 0};
    if (m < p.M && c0 + c < C) {
      if (second) {
        const float s = p.s[m];
        const int8_t* src = p.q + (int64_t)m * p.ldq + c0 + c;
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (c0 + c + e < C) v[e] = (float)src[e] * s;
      } else {
        load8((const T*)p.dy + (int64_t)m * p.lddy, c0 + c, C, v);
      }
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) tile[r][c + e] = from_f32<T>(v[e]);
  }
  __syncthreads();
  T* dst = (T*)(second ? p.xt : p.dyt);
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int c = i * 32 + tid / 8, r0 = (tid % 8) * 8;
    if (c0 + c >= C || m0 + r0 >= p.Mp) continue;  // (Mp is a multiple of 8)
    T o[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) o[e] = tile[r0 + e][c];
    __builtin_memcpy(__builtin_assume_aligned(dst + (int64_t)(c0 + c) * p.Mp + m0 + r0, 16), o, 16);
  }
}

struct Dw8Args {
  NtOperands o;
  void* c;  // direct: [N][ldc]; partial: fp32 [splits][N][K]
  int64_t ldc;
  int m_tiles, n_tiles, splits;
};

template <typename T, int B, int NB, bool PARTIAL>
__global__ __launch_bounds__(512) void dw8_kernel(const Dw8Args p) {
  using G = NtTile<Op16<T>, B, NB>;
  extern __shared__ __align__(16) uint8_t lds[];
  int sp, mt, nt;
  nt_place(p.m_tiles, p.n_tiles, sp, mt, nt);
  const int units = (p.o.K + 127) / 128;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  f32x4 acc[G::TN][G::TM];
  (void)G::run(p.o, lds, mt * B, nt * B, (int)((int64_t)units * sp / p.splits), (int)((int64_t)units * (sp + 1) / p.splits), wave, lane, acc);
  using CT = std::conditional_t<PARTIAL, float, T>;
  CT* c = (CT*)p.c + (PARTIAL ? (int64_t)sp * p.o.M * p.ldc : 0);
  const bool v4 = p.ldc % 4 == 0 && ((uintptr_t)p.c & (4 * sizeof(CT) - 1)) == 0;
  const int M = p.o.M, N = p.o.N, m0 = G::row(mt * B, wave, lane), n0 = G::column(nt * B, wave, lane);
#pragma unroll
  for (int i = 0; i < G::TN; ++i)
#pragma unroll
    for (int j = 0; j < G::TM; ++j) {
      const int m = m0 + 16 * j, n = n0 + 16 * i;
      if (m >= M || n >= N) continue;
      const f32x4 v = acc[i][j];
      CT* dst = c + m * p.ldc + n;
      if (n + 3 < N && v4) {
        store4<CT>(dst, v[0], v[1], v[2], v[3]);
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (n + e < N) dst[e] = from_f32<CT>(v[e]);
      }
    }
}

// Adds the ranges' sums in their order: 4 columns a thread; part [splits][N][ldp], ldp a multiple of 4.
template <typename T>
__global__ __launch_bounds__(256) void dw8_join_kernel(const float* __restrict__ part, int splits, int64_t ldp, T* __restrict__ c,
                                                       int64_t ldc, int N, int K) {
  const int k = (blockIdx.x * 256 + threadIdx.x) * 4, n = blockIdx.y;
  if (k >= K) return;
  const float* src = part + n * ldp + k;
  float4 v = *reinterpret_cast<const float4*>(src);
  for (int i = 1; i < splits; ++i) {
    const float4 q = *reinterpret_cast<const float4*>(src + i * N * ldp);
    v.x += q.x; v.y += q.y; v.z += q.z; v.w += q.w;
  }
  const float o[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int e = 0; e < 4; ++e)
    if (k + e < K) c[n * ldc + k + e] = from_f32<T>(o[e]);
}

// fp32: the kept input itself
__global__ __launch_bounds__(256) void dw8_values_kernel(const int8_t* __restrict__ q, int64_t ldq, const float* __restrict__ s,
                                                         float* __restrict__ x, int K) {
  const int64_t m = blockIdx.y;
  const int k = blockIdx.x * 256 + threadIdx.x;
  if (k < K) x[m * K + k] = (float)q[m * ldq + k] * s[m];
}

struct DwPlan {
  int64_t Mp, dyt_at, xt_at, part_at, ldp, bytes;
  int tile, splits;
};

int64_t up256(int64_t v) { return (v + 255) / 256 * 256; }

DwPlan make_plan(int dt, int64_t M, int64_t N, int64_t K) {
  DwPlan p{};
  if (dt == MLS_F32) {
    p.xt_at = up256(mlsx_dw_fp32_workspace(M, N, K));
    p.bytes = p.xt_at ? p.xt_at + up256(M * K * 4) : 0;
    return p;
  }
  p.Mp = cdiv(M, 8) * 8;
  p.xt_at = up256(N * p.Mp * 2);
  p.part_at = p.xt_at + up256(K * p.Mp * 2);
  p.bytes = p.part_at;
  p.tile = cdiv(N, 256) * cdiv(K, 256) >= 128 ? 256 : 128;
  p.splits = 1;
  if (p.tile == 128) {
    const int64_t tiles = cdiv(N, 128) * cdiv(K, 128), units = cdiv(M, 64);
    p.splits = (int)std::max<int64_t>(1, std::min<int64_t>({512 / tiles, units / 4, 16}));
  }
  if (p.splits > 1) {
    p.ldp = cdiv(K, 4) * 4;
    p.bytes += up256(p.splits * N * p.ldp * 4);
  }
  return p;
}

template <typename T, int B, int NB, bool PARTIAL>
int launch_dw8(const Dw8Args& a, hipStream_t st) {
  const char* fn = "mlsx_dw_int8";
  const int64_t blocks = (int64_t)a.m_tiles * a.n_tiles * a.splits;
  if (blocks > 0x7FFFFFFF) return fail(MLS_ERR_UNSUPPORTED, "%s: %d x %d", fn, a.o.M, a.o.N);
  auto kern = dw8_kernel<T, B, NB, PARTIAL>;
  constexpr int lds = NtTile<Op16<T>, B, NB>::LDS;
  if (lds > 32768 && hipFuncSetAttribute((const void*)kern, hipFuncAttributeMaxDynamicSharedMemorySize, lds) != hipSuccess)
    return fail(MLS_ERR_HIP, "%s: cannot reserve %d bytes of LDS", fn, lds);
  hipLaunchKernelGGL(kern, dim3((unsigned)blocks), dim3(512), lds, st, a);
  return check_launch(fn);
}

template <typename T>
int run16(const void* dy, int64_t lddy, const int8_t* q, int64_t ldq, const float* s, void* dw, int64_t lddw, int64_t M, int64_t N,
          int64_t K, const DwPlan& p, uint8_t* ws, hipStream_t st) {
  const char* fn = "mlsx_dw_int8";
  const TurnArgs t{dy, lddy, q, ldq, s, (int)M, (int)N, (int)K, (int)p.Mp, ws, ws + p.xt_at};
  hipLaunchKernelGGL(dw8_turn_kernel<T>, dim3((unsigned)cdiv(std::max(N, K), 64), (unsigned)cdiv(M, 64), 2), dim3(256), 0, st, t);
  if (const int rc = check_launch(fn)) return rc;
  const int ld = (int)p.Mp * 2;
  Dw8Args a{{ws, ws + p.xt_at, ld, ld, (int)N, (int)K, ld}, dw, lddw, (int)cdiv(N, p.tile), (int)cdiv(K, p.tile), p.splits};
  if (p.splits == 1) return p.tile == 256 ? launch_dw8<T, 256, 2, false>(a, st) : launch_dw8<T, 128, 4, false>(a, st);
  a.c = ws + p.part_at;
  a.ldc = p.ldp;
  if (const int rc = launch_dw8<T, 128, 4, true>(a, st)) return rc;
  hipLaunchKernelGGL(dw8_join_kernel<T>, dim3((unsigned)cdiv(K, 1024), (unsigned)N), dim3(256), 0, st,
                     (const float*)(ws + p.part_at), p.splits, p.ldp, (T*)dw, lddw, (int)N, (int)K);
  return check_launch(fn);
}

}  // namespace

}  // namespace mls

using namespace mls;

extern "C" int64_t mlsx_dw_int8_workspace(int dt, int64_t M, int64_t N, int64_t K) {
  if (M < 1 || N < 1 || K < 1 || M > (1 << 20) || N > (1 << 22) || K > (1 << 22)) return 0;
  return make_plan(dt, M, N, K).bytes;
}

extern "C" int mlsx_dw_int8(const void* dy, int dt, int64_t lddy, const int8_t* q, int64_t ldq, const float* s, void* dw,
                            int64_t lddw, int64_t M, int64_t N, int64_t K, void* ws, int64_t ws_bytes, mls_stream_t stream) {
  const char* fn = "mlsx_dw_int8";
  if (M < 1 || N < 0 || K < 0) return fail(MLS_ERR_ARG, "%s: bad size", fn);
  if (!is_float_dt(dt)) return fail(MLS_ERR_ARG, "%s: bad dtype %d", fn, dt);
  if (N == 0 || K == 0) return MLS_OK;
  const int64_t need = mlsx_dw_int8_workspace(dt, M, N, K);
  if (need == 0) return fail(MLS_ERR_UNSUPPORTED, "%s: M=%lld N=%lld K=%lld", fn, (long long)M, (long long)N, (long long)K);
  if (!dy || !q || !s || !dw || !ws) return fail(MLS_ERR_ARG, "%s: null pointer", fn);
  if (lddy < N || ldq < K || lddw < K) return fail(MLS_ERR_ARG, "%s: bad leading dimension", fn);
  if (ws_bytes < need || !aligned(ws, 16)) return fail(MLS_ERR_ARG, "%s: workspace too small or misaligned", fn);
  const DwPlan p = make_plan(dt, M, N, K);
  const hipStream_t st = (hipStream_t)stream;
  uint8_t* w = (uint8_t*)ws;
  if (dt == MLS_F16) return run16<_Float16>(dy, lddy, q, ldq, s, dw, lddw, M, N, K, p, w, st);
  if (dt == MLS_BF16) return run16<__bf16>(dy, lddy, q, ldq, s, dw, lddw, M, N, K, p, w, st);
  float* x = (float*)(w + p.xt_at);
  if (M > 65535) return fail(MLS_ERR_UNSUPPORTED, "%s: M=%lld", fn, (long long)M);
  hipLaunchKernelGGL(dw8_values_kernel, dim3((unsigned)cdiv(K, 256), (unsigned)M), dim3(256), 0, st, q, ldq, s, x, (int)K);
  if (const int rc = check_launch(fn)) return rc;
  return mlsx_dw_fp32((const float*)dy, lddy, x, K, (float*)dw, lddw, M, N, K, ws, p.xt_at, stream);
}
