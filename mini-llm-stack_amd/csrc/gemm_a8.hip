// y[m][n] = (sum_k xq[m][k] wq[n][k]) sw[n] sx[m] + bias[n]: codes of activations (a scale a row) times INT8
// weights (a scale a row) on the 8-bit matrix cores. The sums are whole numbers of 32 bits and exact, so
// neither tiles nor K ranges nor the order of their joining changes a result.
//
// Three kernels:
//   few rows (a8_few_kernel): bound by reading the weights once (45 MB, from HBM: 13.1 us, 3.4 TB/s); operands go
//     straight to registers, a block of 16 wavefronts shares 16 outputs' weight rows and splits K, and x can be
//     quantized on the way (one row, 4096 -> 4096: 4.8 us);
//   tiles (a8_tile_kernel): both operands staged through LDS by loads that write it directly (nt_tile.h), K split over
//     blocks where the tiles would not fill the GPU;
//   join (a8_join_kernel): adds the K ranges' sums and applies scales and bias.
// From 17 rows: tiles. (Up to 64 rows a tile takes as long as for 64, about 10 us at 4096 -> 4096; 16 rows here 6.3.)
#include <algorithm>

#include "act8.h"
#include "nt_tile.h"

namespace mls {

namespace {

struct Scales {
  const float* sx;
  const void* sw;
  const void* bias;  // null: none
  int sw_dt, bias_dt;
};

__device__ __forceinline__ float float_at(const void* p, int dt, int64_t i) {
  if (dt == MLS_F32) return ((const float*)p)[i];
  if (dt == MLS_F16) return (float)((const _Float16*)p)[i];
  return (float)((const __bf16*)p)[i];
}

// One rounding at each product: a weight's scale first, so that a huge row scale meets a sum that is
// already small.
__device__ __forceinline__ float scaled(int acc, float sw, float sx, float bias) { return (float)acc * sw * sx + bias; }

__device__ __forceinline__ i32x4 mma8(const i32x4& a, const i32x4& b, const i32x4& c) {
  return __builtin_amdgcn_mfma_i32_16x16x64_i8(a, b, c, 0, 0, 0);
}

struct Int8Op {
  using Acc = i32x4;
  __device__ static __forceinline__ i32x4 mma(const i32x4& a, const i32x4& b, const i32x4& c) { return mma8(a, b, c); }
};

// ---------------------------------------------------------------- tiles

struct TileArgs {
  NtOperands o;
  void* c;  // direct: [M][ldc]; partial: int32 [splits][M][N]
  Scales s;
  int64_t ldc;
  int m_tiles, n_tiles, splits;
};

// T: a form of tile (nt_tile.h)
template <typename CT, class T, bool PARTIAL>
__global__ __launch_bounds__(T::THREADS) void a8_tile_kernel(const TileArgs p) {
  extern __shared__ __align__(16) uint8_t lds[];
  int sp, mt, nt;
  nt_place(p.m_tiles, p.n_tiles, sp, mt, nt);
  const int units = (p.o.K + 127) / 128;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  i32x4 acc[T::TN][T::TM];
  if (!T::run(p.o, lds, mt * T::BM, nt * T::BN, (int)((int64_t)units * sp / p.splits), (int)((int64_t)units * (sp + 1) / p.splits), wave,
              lane, acc))
    return;
  const int M = p.o.M, N = p.o.N, m0 = T::row(mt * T::BM, wave, lane), n0 = T::column(nt * T::BN, wave, lane);
  if constexpr (PARTIAL) {
#pragma unroll
    for (int i = 0; i < T::TN; ++i)
#pragma unroll
      for (int j = 0; j < T::TM; ++j) {
        const int m = m0 + 16 * j, n = n0 + 16 * i;
        if (m >= M || n >= N) continue;
        const i32x4 v = acc[i][j];
        int* dst = (int*)p.c + ((int64_t)sp * M + m) * N + n;
        if (n + 3 < N && N % 4 == 0) {
          *reinterpret_cast<int4*>(dst) = make_int4(v[0], v[1], v[2], v[3]);
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (n + e < N) dst[e] = v[e];
        }
      }
    return;
  }
  // all scales before the first store, which they would otherwise wait for one by one
  float sx[T::TM], sw[T::TN][4], bias[T::TN][4];
#pragma unroll
  for (int j = 0; j < T::TM; ++j) sx[j] = p.s.sx[min(m0 + 16 * j, M - 1)];
#pragma unroll
  for (int i = 0; i < T::TN; ++i)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int n = min(n0 + 16 * i + e, N - 1);
      sw[i][e] = float_at(p.s.sw, p.s.sw_dt, n);
      bias[i][e] = p.s.bias ? float_at(p.s.bias, p.s.bias_dt, n) : 0.0f;
    }
  const bool wide = (p.ldc * sizeof(CT)) % 16 == 0 && ((uintptr_t)p.c & 15) == 0;
  if constexpr (sizeof(CT) == 2) {
    const int lk = lane >> 4, nt0 = n0 - 4 * lk;
#pragma unroll
    for (int i = 0; i < T::TN; i += 2)
#pragma unroll
      for (int j = 0; j < T::TM; ++j) {
        uint2 o[2];
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          CT y[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) y[e] = from_f32<CT>(scaled(acc[i + t][j][e], sw[i + t][e], sx[j], bias[i + t][e]));
          o[t] = make_uint2(pack2_bits(y[0], y[1]), pack2_bits(y[2], y[3]));
        }
        const int m = m0 + 16 * j;
        nt_store_pair((uint16_t*)p.c + (int64_t)m * p.ldc + nt0 + 16 * i, nt0 + 16 * i, N, o[0], o[1], lk, m < M, wide);
      }
  } else {
#pragma unroll
    for (int i = 0; i < T::TN; ++i)
#pragma unroll
      for (int j = 0; j < T::TM; ++j) {
        const int m = m0 + 16 * j, n = n0 + 16 * i;
        if (m >= M || n >= N) continue;
        CT* dst = (CT*)p.c + (int64_t)m * p.ldc + n;
        float y[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) y[e] = scaled(acc[i][j][e], sw[i][e], sx[j], bias[i][e]);
        if (n + 3 < N && wide) {
          store4<CT>(dst, y[0], y[1], y[2], y[3]);
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (n + e < N) dst[e] = from_f32<CT>(y[e]);
        }
      }
  }
}

// Adds the K ranges' sums: 4 columns a thread.
template <typename CT>
__global__ __launch_bounds__(256) void a8_join_kernel(const int* __restrict__ part, int splits, CT* __restrict__ c, int64_t ldc,
                                                      Scales s, int M, int N) {
  const int n = (blockIdx.x * 256 + threadIdx.x) * 4, m = blockIdx.y;
  if (n >= N) return;
  const int64_t step = (int64_t)M * N;
  const int* src = part + (int64_t)m * N + n;
  int v[4] = {0, 0, 0, 0};
  if (N % 4 == 0) {
    for (int i = 0; i < splits; ++i) {
      const int4 q = *reinterpret_cast<const int4*>(src + i * step);
      v[0] += q.x; v[1] += q.y; v[2] += q.z; v[3] += q.w;
    }
  } else {
    for (int i = 0; i < splits; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (n + e < N) v[e] += src[i * step + e];
  }
  const float sx = s.sx[m];
#pragma unroll
  for (int e = 0; e < 4; ++e)
    if (n + e < N)
      c[(int64_t)m * ldc + n + e] =
          from_f32<CT>(scaled(v[e], float_at(s.sw, s.sw_dt, n + e), sx, s.bias ? float_at(s.bias, s.bias_dt, n + e) : 0.0f));
}

// ---------------------------------------------------------------- few rows

struct FewArgs {
  const void* x;  // codes, or values to quantize
  const uint8_t* w;
  void* c;
  Scales s;
  int64_t ldx, ldc;
  int ldw;
  int M, N, K;
  int values;  // columns of x to quantize, a multiple of 8 (K: those and the weights' padding)
};

constexpr int kFewWaves = 16;

// One block: outputs n0 .. n0 + 15 of all M <= 16 rows; wavefront i takes every 16th step of 128 k. Lane
// (lr, lk) holds 32 consecutive bytes of weight row lr a step, two operands; a step's k order is that of both operands
// alike. XT: the type that x is quantized from on the way, int8_t: codes.
//
// Quantizing: 16 / R wavefronts a row (R: M rounded up to a power of two), C chunks of 8 values a lane, the codes
// in LDS for all wavefronts. Every block repeats it, while its first weights are on their way: one launch
// instead of two.
template <typename XT, typename CT, int C>
__global__ __launch_bounds__(64 * kFewWaves) void a8_few_kernel(const FewArgs p) {
  constexpr bool CODES = __is_same(XT, int8_t);
  extern __shared__ __align__(16) uint8_t codes[];  // [M][ldq]
  __shared__ __align__(16) int sums[kFewWaves][64][4];
  __shared__ uint32_t tops[kFewWaves];
  __shared__ float scales[16];

  constexpr int U = 2;  // steps in flight
  const int n0 = blockIdx.x * 16;
  const int lane = threadIdx.x & 63, lr = lane & 15, lk = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const __amdgpu_buffer_rsrc_t rsw = nt_rows(p.w, n0, p.ldw, min(16, p.N - n0), p.K);
  const int steps = (p.K + 127) / 128;
  const int w_off = lr * p.ldw + lk * 32;

  uint4 wv[U][2];
  auto load_w = [&](int step) __attribute__((always_inline)) {
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int h = 0; h < 2; ++h)  // (past the operand: zeros)
        wv[u][h] = __builtin_bit_cast(uint4, __builtin_amdgcn_raw_buffer_load_b128(rsw, w_off + (step + u * kFewWaves) * 128 + h * 16, 0, 0));
  };

  const int ldq = (p.K + 127) / 128 * 128 + 16;
  if constexpr (!CODES) {
    int R = 1;
    while (R < p.M) R *= 2;
    const int P = kFewWaves / R, row = wave / P, part = wave % P;
    // (no branch around a load: its merge would wait for the weights in flight)
    const XT* src = (const XT*)p.x + min(row, p.M - 1) * p.ldx;
    Raw8<XT> raw[C];
#pragma unroll
    for (int c = 0; c < C; ++c) raw[c] = fetch8(src, ((c * P + part) * 64 + lane) * 8, p.values);
    // x of all wavefronts before any weights, behind which the last would get it
    __builtin_amdgcn_sched_barrier(0);
    asm volatile("s_barrier" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
    load_w(wave);
    __builtin_amdgcn_sched_barrier(0);
    float v[C][8];
    uint32_t top = 0;
#pragma unroll
    for (int c = 0; c < C; ++c) {
      widen8(raw[c], ((c * P + part) * 64 + lane) * 8 < p.values, v[c]);
      top = max(top, max_abs8(v[c]));
    }
    top = group_max_bits<64>(top);
    if (lane == 0) tops[wave] = top;
    __syncthreads();
    if (row < p.M) {
      for (int i = 0; i < P; ++i) top = max(top, tops[row * P + i]);
      const Scale8 g = scale8(top);
      if (part == 0 && lane == 0) scales[row] = g.s;
#pragma unroll
      for (int c = 0; c < C; ++c) {
        const int k = ((c * P + part) * 64 + lane) * 8;
        if (k < ldq - 16) *reinterpret_cast<uint2*>(codes + row * ldq + k) = codes8(v[c], g);
      }
    }
    __syncthreads();
  } else {
    load_w(wave);
  }

  i32x4 acc = i32x4{0, 0, 0, 0};
  const __amdgpu_buffer_rsrc_t rsx =
      CODES ? nt_rows(p.x, 0, p.ldx, p.M, p.K) : nt_rows(p.w, 0, 0, 1, 0);  // (quantized on the way: not used)
  const int x_off = lr * (int)p.ldx + lk * 32;
  for (int step = wave; step < steps; step += U * kFewWaves) {
    uint4 xv[U][2];
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int k = (step + u * kFewWaves) * 128 + lk * 32 + h * 16;
        if constexpr (CODES) {
          // rows past M and columns past K: zeros
          xv[u][h] = __builtin_bit_cast(uint4, __builtin_amdgcn_raw_buffer_load_b128(
                                                   rsx, k < p.K && lr < p.M ? x_off + (step + u * kFewWaves) * 128 + h * 16 : kNtOutside, 0, 0));
        } else {
          xv[u][h] = lr < p.M && k < ldq - 16 ? *reinterpret_cast<const uint4*>(codes + lr * ldq + k) : make_uint4(0, 0, 0, 0);
        }
      }
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int h = 0; h < 2; ++h) acc = mma8(__builtin_bit_cast(i32x4, wv[u][h]), __builtin_bit_cast(i32x4, xv[u][h]), acc);
    if (step + U * kFewWaves < steps) load_w(step + U * kFewWaves);
  }
  *reinterpret_cast<int4*>(sums[wave][lane]) = make_int4(acc[0], acc[1], acc[2], acc[3]);
  __syncthreads();
  const int t = threadIdx.x, m = t / 16, n = n0 + t % 16;
  if (m >= min(p.M, 16) || n >= p.N) return;
  int total = 0;
#pragma unroll
  for (int i = 0; i < kFewWaves; ++i) total += sums[i][t % 16 / 4 * 16 + m][t % 4];
  const float sx = CODES ? p.s.sx[m] : scales[m];
  ((CT*)p.c)[m * p.ldc + n] =
      from_f32<CT>(scaled(total, float_at(p.s.sw, p.s.sw_dt, n), sx, p.s.bias ? float_at(p.s.bias, p.s.bias_dt, n) : 0.0f));
}

// Chunks of 8 values a lane that quantizing M rows of K takes in a few-rows block.
int few_chunks(int64_t M, int64_t K) {
  int64_t R = 1;
  while (R < M) R *= 2;
  return (int)cdiv(cdiv(K, 128) * 16, 64 * (kFewWaves / R));
}

// ---------------------------------------------------------------- host

struct Plan {
  bool few, fused;        // the kernel for few rows; which quantizes x itself
  bool pad_w, own_x;      // operands copied (or codes made) into the workspace
  int64_t kpad;
  int form, splits;       // of kNtForms; K ranges
  int64_t x_at, s_at, w_at, part_at, bytes;
};

int64_t up256(int64_t v) { return (v + 255) / 256 * 256; }

bool rows_fit(const void* p, int64_t ld, int64_t K) {
  return K % 16 == 0 && ld % 16 == 0 && aligned(p, 16) && ld < (1 << 22);
}

Plan make_plan(const mlsx_a8w8_args& a) {
  Plan p{};
  const bool codes = a.x_dt < 0;
  p.kpad = (a.K + 127) / 128 * 128;  // (rows of whole cache lines: 20% off a stage's loads against rows 64 bytes apart)
  p.pad_w = !rows_fit(a.w, a.ldw, a.K);
  p.few = a.M <= 16;
  // A block's quantizing takes about 0.25 us a chunk, in every round of blocks; a launch of its own 3 us (in one launch and in two:
  // 4 rows of 11008 -> 4096, 6 chunks, 14.2 and 17.7 us; 8 of 4096 -> 4096, 4 chunks, 6.1 and 9.3; 16 of 4096 -> 11008, 8 chunks, 26.4 and 17.6)
  p.fused = a.x_dt == a.c_dt && p.few && a.K % 8 == 0 && few_chunks(a.M, a.K) <= 6 && few_chunks(a.M, a.K) * cdiv(a.N, 4096) <= 6;
  p.own_x = codes ? !rows_fit(a.x, a.ldx, a.K) : !p.fused;
  p.splits = 1;
  if (!p.few) nt_choose(a.M, a.N, a.K, p.form, p.splits);
  int64_t at = 0;
  if (p.own_x) {
    p.x_at = at;
    at += up256(a.M * p.kpad);
    p.s_at = at;
    if (!codes) at += up256(a.M * 4);
  }
  if (p.pad_w) {
    p.w_at = at;
    at += up256(a.N * p.kpad);
  }
  if (p.splits > 1) {
    p.part_at = at;
    at += up256(p.splits * a.M * a.N * 4);
  }
  p.bytes = at;
  return p;
}

template <typename CT, class T, bool PARTIAL>
int launch_tiles(TileArgs t, hipStream_t st) {
  t.m_tiles = (int)cdiv(t.o.M, T::BM);
  t.n_tiles = (int)cdiv(t.o.N, T::BN);
  const int64_t blocks = (int64_t)t.m_tiles * t.n_tiles * t.splits;
  if (!grid_fits(blocks, T::THREADS)) return fail(MLS_ERR_UNSUPPORTED, "a8w8: %d x %d", t.o.M, t.o.N);
  auto kern = a8_tile_kernel<CT, T, PARTIAL>;
  constexpr int lds = T::LDS;
  // (a call a launch: the limit is the function's on the current device)
  if (lds > 32768 && hipFuncSetAttribute((const void*)kern, hipFuncAttributeMaxDynamicSharedMemorySize, lds) != hipSuccess)
    return fail(MLS_ERR_HIP, "a8w8: cannot reserve %d bytes of LDS", lds);
  hipLaunchKernelGGL(kern, dim3((unsigned)blocks), dim3(T::THREADS), lds, st, t);
  return check_launch("a8w8");
}

template <typename CT, class T>
int launch_tile(TileArgs t, void* part, hipStream_t st) {
  if constexpr (T::RANGES) {
    if (t.splits > 1) {
      void* c = t.c;
      t.c = part;
      if (const int rc = launch_tiles<CT, T, true>(t, st)) return rc;
      hipLaunchKernelGGL(a8_join_kernel<CT>, dim3((unsigned)cdiv(t.o.N, 1024), (unsigned)t.o.M), dim3(256), 0, st, (const int*)part,
                         t.splits, (CT*)c, t.ldc, t.s, t.o.M, t.o.N);
      return check_launch("a8w8 (join)");
    }
  }
  return launch_tiles<CT, T, false>(t, st);
}

template <typename XT, typename CT, int C>
int launch_few(const FewArgs& f, hipStream_t st) {
  auto kern = a8_few_kernel<XT, CT, C>;
  const size_t lds = C ? (size_t)f.M * (cdiv(f.K, 128) * 128 + 16) : 0;
  if (lds > 32768 && hipFuncSetAttribute((const void*)kern, hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds) != hipSuccess)
    return fail(MLS_ERR_HIP, "a8w8: cannot reserve %zu bytes of LDS", lds);
  hipLaunchKernelGGL(kern, dim3((unsigned)cdiv(f.N, 16)), dim3(64 * kFewWaves), lds, st, f);
  return check_launch("a8w8 (few rows)");
}

template <typename T>
int launch_fused(const FewArgs& f, int chunks, hipStream_t st) {
  if (chunks <= 1) return launch_few<T, T, 1>(f, st);
  if (chunks <= 2) return launch_few<T, T, 2>(f, st);
  if (chunks <= 4) return launch_few<T, T, 4>(f, st);
  return launch_few<T, T, 6>(f, st);
}

template <typename CT>
int run(const mlsx_a8w8_args& a, const Plan& p, uint8_t* ws, hipStream_t st) {
  const bool codes = a.x_dt < 0;
  const uint8_t* x = (const uint8_t*)a.x;
  const uint8_t* w = (const uint8_t*)a.w;
  int64_t ldx = a.ldx, ldw = a.ldw, K = a.K;
  Scales s{a.sx, a.sw, a.bias, (int)a.sw_dt, (int)a.bias_dt};
  PadRows px{}, pw{};
  if (p.own_x) {
    x = ws + p.x_at;
    ldx = p.kpad;
    if (codes) {
      px = {(const uint8_t*)a.x, a.ldx, a.M, ws + p.x_at};
    } else {
      s.sx = (float*)(ws + p.s_at);
      if (const int rc = launch_quantize_rows(a.x, (int)a.x_dt, a.ldx, a.M, a.K, p.kpad, (int8_t*)(ws + p.x_at), p.kpad,
                                              (float*)(ws + p.s_at), st))
        return rc;
    }
  }
  if (p.pad_w) {
    w = ws + p.w_at;
    ldw = p.kpad;
    pw = {(const uint8_t*)a.w, a.ldw, a.N, ws + p.w_at};
  }
  if (const int rc = launch_pad_rows(px, pw, a.K, p.kpad, st)) return rc;
  // Padded operands: the products of the padding are zeros. (A K that is no multiple of 16 pads both; a quantizing block
  // pads its codes itself.)
  if ((p.own_x || p.fused) && p.pad_w) K = p.kpad;
  if (p.few) {
    FewArgs f{x, w, a.c, s, ldx, a.ldc, (int)ldw, (int)a.M, (int)a.N, (int)K, 0};
    if (!p.fused) return launch_few<int8_t, CT, 0>(f, st);
    f.x = a.x;
    f.ldx = a.ldx;
    f.values = (int)a.K;
    return launch_fused<CT>(f, few_chunks(a.M, a.K), st);
  }
  TileArgs t{{x, w, (int)ldx, (int)ldw, (int)a.M, (int)a.N, (int)K}, a.c, s, a.ldc, 0, 0, p.splits};
  return nt_form<Int8Op>(p.form, [&](auto form) { return launch_tile<CT, typename decltype(form)::type>(t, ws + p.part_at, st); });
}

int check_args(const mlsx_a8w8_args& a, const char* fn) {
  if (a.M < 0 || a.N < 0 || a.K < 1) return fail(MLS_ERR_ARG, "%s: bad size M = %lld, N = %lld, K = %lld", fn, (long long)a.M, (long long)a.N, (long long)a.K);
  if ((a.x_dt >= 0 && !is_float_dt((int)a.x_dt)) || !is_float_dt((int)a.c_dt) || (a.sw_dt != MLS_F32 && a.sw_dt != MLS_F16) ||
      (a.bias && !is_float_dt((int)a.bias_dt)))
    return fail(MLS_ERR_ARG, "%s: bad dtype", fn);
  if (a.K > 131071) return fail(MLS_ERR_UNSUPPORTED, "%s: K = %lld: sums of 131072 products of -128 by -128 pass 32 bits", fn, (long long)a.K);
  if (a.M > (1 << 22) || a.N > (1 << 22)) return fail(MLS_ERR_UNSUPPORTED, "%s: M = %lld, N = %lld", fn, (long long)a.M, (long long)a.N);
  if (a.M == 0 || a.N == 0) return MLS_OK;
  if (!a.c || !a.sw || !a.x || !a.w || (a.x_dt < 0 && !a.sx)) return fail(MLS_ERR_ARG, "%s: null pointer", fn);
  if (a.ldx < a.K || a.ldw < a.K || a.ldc < a.N) return fail(MLS_ERR_ARG, "%s: bad leading dimension", fn);
  return MLS_OK;
}

}  // namespace

}  // namespace mls

using namespace mls;

extern "C" int64_t mlsx_a8w8_ws(const mlsx_a8w8_args* args) {
  if (!args || args->M <= 0 || args->N <= 0 || args->K < 1 || args->K > 131071 || args->M > (1 << 22) || args->N > (1 << 22)) return 0;
  return make_plan(*args).bytes;
}

extern "C" int mlsx_a8w8_form(const mlsx_a8w8_args* args) {
  if (!args || args->M <= 0 || args->N <= 0 || args->K < 1 || args->K > 131071 || args->M > (1 << 22) || args->N > (1 << 22)) return -1;
  const Plan p = make_plan(*args);
  return p.few ? (p.fused ? 1 : 0) : 16 * (p.form + 1) + p.splits;
}

extern "C" int64_t mlsx_a8w8(const mlsx_a8w8_args* args, void* ws, int64_t ws_bytes, mls_stream_t stream) {
  const char* fn = "mlsx_a8w8";
  if (!args) return fail(MLS_ERR_ARG, "%s: null pointer", fn);
  if (const int rc = check_args(*args, fn)) return rc;
  if (args->M == 0 || args->N == 0) return MLS_OK;
  const Plan p = make_plan(*args);
  if (p.bytes && !ws && ws_bytes == 0) return p.bytes;
  if (p.bytes > ws_bytes || (p.bytes && (!ws || !aligned(ws, 16)))) return fail(MLS_ERR_ARG, "%s: workspace too small or misaligned", fn);
  const hipStream_t st = (hipStream_t)stream;
  if (args->c_dt == MLS_F32) return run<float>(*args, p, (uint8_t*)ws, st);
  if (args->c_dt == MLS_F16) return run<_Float16>(*args, p, (uint8_t*)ws, st);
  return run<__bf16>(*args, p, (uint8_t*)ws, st);
}
