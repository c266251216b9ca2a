// Attention of new tokens over a paged K/V cache with grouped heads, on the matrix cores: the
// kernels (paged_gqa.hip says what they compute and which calls take which). Instantiated per
// element type in paged_gqa_f32.hip, paged_gqa_f16.hip and paged_gqa_bf16.hip.
//
// A K/V head's query rows are packed: row r of a sequence is its new token r / group, query head
// r % group of the K/V head's group, so every row of a tile multiplies the same keys. With 16x16
// MFMAs, S^T = K Q^T: a lane holds the scores of one row (lane & 15) for the keys
// 16 a + 4 (lane >> 4) + i. These registers are, as they are, the B operand of
// O^T += V^T P^T over 32 keys (16 in fp32), if the A operand takes V's keys in the same order:
// P never crosses lanes and never sees LDS. K and V tiles arrive by 16-byte loads straight into
// LDS, chunks swizzled by row; V's fragments are read transposed (ds_read_b64_tr_b16).
//
// Softmax with a lazy maximum: m is a row's reference, any value within 2^8 of what the row has
// seen; only a tile with a score above m + 8 (in log2 units) reduces the maximum over lanes and
// rescales l and O. l is a per-lane partial sum until the end. All statistics are fp32. P is
// rounded to the inputs' type for the product with V (half a step, unbiased), l sums it unrounded.
#pragma once

#include <atomic>

#include "common.h"
#include "paged_gqa_args.h"

namespace mls {

typedef short s16x4 __attribute__((ext_vector_type(4)));

// 16 bytes of zeros: what a lane loads for a key outside its range, of a block id outside the
// pool, or for elements past the head dim.
static __device__ __align__(16) const uint32_t gqa_zeros[4] = {0, 0, 0, 0};

template <typename T>
struct GqaType {
  static constexpr bool F32 = sizeof(T) == 4;
  static constexpr int CE = 16 / (int)sizeof(T);  // elements of a 16-byte chunk
  static constexpr int PK = F32 ? 16 : 32;        // keys of one P V product
  // fp16: P is stored times 2^8, so that weights down to 2^-32 of the row's reference keep bits
  static constexpr float OFF = __is_same(T, _Float16) ? 8.0f : 0.0f;
  static constexpr float SLACK = __is_same(T, _Float16) ? 7.0f : 8.0f;
};

// c += A B over one 16-byte chunk per lane: 32 elements of the reduction (16-bit), 16 (fp32)
template <typename T>
__device__ __forceinline__ f32x4 gqa_mma(const uint4& a, const uint4& b, f32x4 c) {
  if constexpr (__is_same(T, __bf16)) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  } else if constexpr (__is_same(T, _Float16)) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  } else {
    c = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(a.x), __uint_as_float(b.x), c, 0, 0, 0);
    c = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(a.y), __uint_as_float(b.y), c, 0, 0, 0);
    c = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(a.z), __uint_as_float(b.z), c, 0, 0, 0);
    return __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(a.w), __uint_as_float(b.w), c, 0, 0, 0);
  }
}

template <typename T>
__device__ __forceinline__ uint32_t gqa_pack2(float lo, float hi) {
  return pack2_bits(from_f32<T>(lo), from_f32<T>(hi));
}

__device__ __forceinline__ void gqa_lds_load16(const void* g, void* lds) {
  __builtin_amdgcn_global_load_lds((__attribute__((address_space(1))) void*)g,
                                   (__attribute__((address_space(3))) void*)lds, 16, 0, 0);
}

// Maximum over the four 16-lane rows of a wavefront, lane & 15 kept apart.
__device__ __forceinline__ float gqa_row_max(float v) {
  v = fmaxf(v, __shfl_xor(v, 16, 64));
  return fmaxf(v, __shfl_xor(v, 32, 64));
}
__device__ __forceinline__ float gqa_row_sum(float v) {
  v += __shfl_xor(v, 16, 64);
  return v + __shfl_xor(v, 32, 64);
}

// Geometry of a tile of BN keys in LDS: rows of DL elements (a power of two), CPR chunks a row.
// Chunk c of K row r sits at c ^ (r & 7); of V row r at c ^ 2 (r & 7) (16-bit: the four rows that
// one group of 16 lanes reads transposed, 32 bytes of each, lie in different banks) or, fp32,
// c ^ 4 ((r >> 2) & 3) (four lane groups read 64 bytes of rows 4 apart).
template <typename T, int DP>
struct GqaTile {
  static constexpr int CE = GqaType<T>::CE;
  static constexpr int DL = DP <= 64 ? 64 : DP <= 128 ? 128 : 256;
  static constexpr int CPR = DL / CE, ROWB = DL * (int)sizeof(T);
  __device__ static __forceinline__ int swz_k(int r) { return r & 7; }
  __device__ static __forceinline__ int swz_v(int r) {
    if constexpr (GqaType<T>::F32) return ((r >> 2) & 3) << 2;
    return (r << 1) & (CPR >= 16 ? 14 : 6);
  }
};

// Loads the K and V rows of BN keys into LDS. Every wavefront finds the place of every key (lane i:
// key i), THREADS of them share the loads. `off`: byte offset of key `lane` in the pools, -1 for a
// key to be read as zeros. wave: which of the THREADS / 64 this is.
template <typename T, int DP, int BN, int THREADS, bool VEC>
__device__ __forceinline__ void gqa_fill(uint8_t* kt, uint8_t* vt, const uint8_t* kbase, const uint8_t* vbase, int64_t off,
                                         int D, int wave, int lane) {
  using G = GqaTile<T, DP>;
  constexpr int ITER = BN * G::CPR / THREADS, RPI = THREADS / G::CPR;  // rows an instruction of all threads
  static_assert(BN <= 64 && ITER * THREADS == BN * G::CPR, "whole instructions");
  const int slot = wave * 64 + lane;
#pragma unroll
  for (int u = 0; u < ITER; ++u) {
    const int row = RPI > 0 ? u * RPI + slot / G::CPR : (u * THREADS + slot) / G::CPR;
    const int c = slot % G::CPR;
    const int lo = __shfl((int)off, row, 64), hi = __shfl((int)(off >> 32), row, 64);
    const int64_t o = ((int64_t)hi << 32) | (uint32_t)lo;
    const int ck = c ^ G::swz_k(row), cv = c ^ G::swz_v(row);
    uint8_t* kd = kt + (u * THREADS + wave * 64) * 16;
    uint8_t* vd = vt + (u * THREADS + wave * 64) * 16;
    if constexpr (VEC) {
      const uint8_t* zero = reinterpret_cast<const uint8_t*>(gqa_zeros);
      gqa_lds_load16(hi >= 0 && ck * G::CE < D ? kbase + o + ck * 16 : zero, kd);
      gqa_lds_load16(hi >= 0 && cv * G::CE < D ? vbase + o + cv * 16 : zero, vd);
    } else {
      T kx[G::CE], vx[G::CE];
#pragma unroll
      for (int e = 0; e < G::CE; ++e) {
        const int dk = ck * G::CE + e, dv = cv * G::CE + e;
        kx[e] = hi >= 0 && dk < D ? reinterpret_cast<const T*>(kbase + o)[dk] : (T)0.0f;
        vx[e] = hi >= 0 && dv < D ? reinterpret_cast<const T*>(vbase + o)[dv] : (T)0.0f;
      }
      *reinterpret_cast<uint4*>(kd + lane * 16) = __builtin_bit_cast(uint4, kx);
      *reinterpret_cast<uint4*>(vd + lane * 16) = __builtin_bit_cast(uint4, vx);
    }
  }
}

// The place of key `key` in the pools (bytes from a head's base), from its block id.
__device__ __forceinline__ int64_t gqa_key_offset(const GqaArgs& a, int key, int blk, bool in, int esz) {
  const bool ok = in && blk >= 0 && blk < a.num_blocks;
  const int t = key - gqa_block_of(a, key) * a.BS;
  return ok ? ((int64_t)blk * a.kv_sb + (int64_t)t * a.kv_st) * esz : -1;
}

// One wavefront's rows: 16 NT query rows with their softmax state.
template <typename T, int DP, int NT>
struct GqaRows {
  using G = GqaTile<T, DP>;
  using K = GqaType<T>;
  static constexpr int QT = DP / (4 * K::CE), OT = DP / 16;
  uint4 q[NT][QT];
  f32x4 o[NT][OT];
  float m[NT], l[NT];
  int lo[NT], hi[NT], pos[NT];  // the keys that a row sees: [lo, hi)
  float slope[NT];              // times log2(e)
  int lo_min, lo_max, hi_min, hi_max;  // over the wavefront's rows

  // row0: the wavefront's first packed row of the tile's sequence
  __device__ __forceinline__ void init(const GqaArgs& a, const GqaPlan& p, int row0, int kvh, int lane) {
    const int g = lane >> 4;
    lo_min = hi_min = 0x7FFFFFFF;
    lo_max = hi_max = -0x7FFFFFFF;
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      m[n] = -3.402823466e38f;
      l[n] = 0.0f;
#pragma unroll
      for (int d = 0; d < OT; ++d) o[n][d] = f32x4{0.f, 0.f, 0.f, 0.f};
      const int r = row0 + 16 * n + (lane & 15);
      const bool in = r < p.rows;
      const int tok = min(p.tok0 + r / a.group, a.T - 1), head = kvh * a.group + r % a.group;
      gqa_row_range(a, p, tok, lo[n], hi[n], pos[n]);
      if (in) {
        lo_min = min(lo_min, lo[n]);
        lo_max = max(lo_max, lo[n]);
        hi_min = min(hi_min, hi[n]);
        hi_max = max(hi_max, hi[n]);
      }
      slope[n] = a.slopes ? a.slopes[head] * 1.44269504f : 0.0f;
      const T* src = static_cast<const T*>(a.q) + tok * a.q_st + head * a.q_sh;
#pragma unroll
      for (int t = 0; t < QT; ++t) {
        const int d0 = (4 * t + g) * K::CE;
        uint4 v = make_uint4(0, 0, 0, 0);
        if (a.q_vec) {
          if (in && d0 < a.D) v = *reinterpret_cast<const uint4*>(src + d0);
        } else {
          T x[K::CE];
#pragma unroll
          for (int e = 0; e < K::CE; ++e) x[e] = in && d0 + e < a.D ? src[d0 + e] : (T)0.0f;
          v = __builtin_bit_cast(uint4, x);
        }
        q[n][t] = v;
      }
    }
#pragma unroll
    for (int off = 1; off < 16; off <<= 1) {
      lo_min = min(lo_min, __shfl_xor(lo_min, off, 64));
      lo_max = max(lo_max, __shfl_xor(lo_max, off, 64));
      hi_min = min(hi_min, __shfl_xor(hi_min, off, 64));
      hi_max = max(hi_max, __shfl_xor(hi_max, off, 64));
    }
    lo_min = __builtin_amdgcn_readfirstlane(lo_min);
    lo_max = __builtin_amdgcn_readfirstlane(lo_max);
    hi_min = __builtin_amdgcn_readfirstlane(hi_min);
    hi_max = __builtin_amdgcn_readfirstlane(hi_max);
  }

  // Whether every row of the wavefront sees all of the keys [j, j + n), and whether any row sees any
  __device__ __forceinline__ bool sees_all(int j, int n) const { return lo_max <= j && j + n <= hi_min; }
  __device__ __forceinline__ bool sees_any(int j, int n) const { return lo_min < j + n && j < hi_max; }

  // The keys [j0, j0 + BN) in kt / vt; okmask: the keys that are there at all.
  template <int BN>
  __device__ __forceinline__ void step(const GqaArgs& a, const uint8_t* kt, const uint8_t* vt, int j0, uint64_t okmask,
                                       int lane) {
    constexpr int KT = BN / 16;
    const int g = lane >> 4, c = lane & 15;
    f32x4 s[NT][KT];
#pragma unroll
    for (int k = 0; k < KT; ++k) {
#pragma unroll
      for (int n = 0; n < NT; ++n) s[n][k] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int t = 0; t < QT; ++t) {
        const int row = 16 * k + c;
        const uint4 kf = *reinterpret_cast<const uint4*>(kt + row * G::ROWB + (((4 * t + g) ^ G::swz_k(row)) << 4));
#pragma unroll
        for (int n = 0; n < NT; ++n) s[n][k] = gqa_mma<T>(kf, q[n][t], s[n][k]);
      }
    }
    // scores in log2 units: s * cc
    float cc = a.c;
    if (!a.simple) {
      cc = 1.0f;
      scored<KT>(a, s, j0, g);
    }
    constexpr uint64_t FULL = BN == 64 ? ~0ull : (1ull << (BN & 63)) - 1;
    const bool masked = okmask != FULL || !sees_all(j0, BN);
    if (masked) {
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int k = 0; k < KT; ++k)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int kk = 16 * k + 4 * g + i, j = j0 + kk;
            const bool see = lo[n] <= j && j < hi[n] && ((okmask >> kk) & 1);
            s[n][k][i] = see ? s[n][k][i] : -__builtin_huge_valf();
          }
    }
    float mx[NT];
    bool over = false;
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      mx[n] = s[n][0][0];
#pragma unroll
      for (int k = 0; k < KT; ++k)
#pragma unroll
        for (int i = 0; i < 4; ++i) mx[n] = fmaxf(mx[n], s[n][k][i]);
      mx[n] *= cc;
      over = over || mx[n] > m[n] + (K::OFF + K::SLACK);
    }
    if (__any(over)) {
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        const float mn = fmaxf(m[n], gqa_row_max(mx[n]) - K::OFF);
        const float f = __builtin_amdgcn_exp2f(m[n] - mn);
        m[n] = mn;
        l[n] *= f;
#pragma unroll
        for (int d = 0; d < OT; ++d) o[n][d] *= f;
      }
    }
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int k = 0; k < KT; ++k)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          s[n][k][i] = __builtin_amdgcn_exp2f(fmaf(s[n][k][i], cc, -m[n]));
          l[n] += s[n][k][i];
        }
    product<BN>(s, vt, g, c);
  }

  // Raw products -> scores in log2 units, with the cap and the bias by distance
  template <int KT>
  __device__ __forceinline__ void scored(const GqaArgs& a, f32x4 (&s)[NT][KT], int j0, int g) const {
    if (a.cap > 0.0f) {
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int k = 0; k < KT; ++k)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float y = s[n][k][i] * a.to_cap;  // scale / cap
            // 1 - 2 / (e^2y + 1) is off by 2^-23 of the cap: too much for fp32 scores only
            float t;
            if constexpr (K::F32) t = tanhf(y);
            else t = 1.0f - 2.0f * __builtin_amdgcn_rcpf(__builtin_amdgcn_exp2f(y * 2.88539008f) + 1.0f);
            s[n][k][i] = t * a.cap;  // cap log2(e)
          }
    } else {
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int k = 0; k < KT; ++k) s[n][k] *= a.c;
    }
    if (a.slopes) {
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int k = 0; k < KT; ++k)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            s[n][k][i] = fmaf(-slope[n], fabsf((float)(pos[n] - (j0 + 16 * k + 4 * g + i))), s[n][k][i]);
    }
  }

  // O^T += V^T P^T
  template <int BN>
  __device__ __forceinline__ void product(const f32x4 (&s)[NT][BN / 16], const uint8_t* vt, int g, int c) {
    if constexpr (K::F32) {
#pragma unroll
      for (int k = 0; k < BN / 16; ++k)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int row = 16 * k + 4 * g + i;
#pragma unroll
          for (int d = 0; d < OT; ++d) {
            const int ch = (4 * d + (c >> 2)) ^ G::swz_v(row);
            const float v = *reinterpret_cast<const float*>(vt + row * G::ROWB + ch * 16 + (c & 3) * 4);
#pragma unroll
            for (int n = 0; n < NT; ++n) o[n][d] = __builtin_amdgcn_mfma_f32_16x16x4f32(v, s[n][k][i], o[n][d], 0, 0, 0);
          }
        }
    } else {
#pragma unroll
      for (int h = 0; h < BN / 32; ++h) {
        uint4 pf[NT];
#pragma unroll
        for (int n = 0; n < NT; ++n)
          pf[n] = make_uint4(gqa_pack2<T>(s[n][2 * h][0], s[n][2 * h][1]), gqa_pack2<T>(s[n][2 * h][2], s[n][2 * h][3]),
                             gqa_pack2<T>(s[n][2 * h + 1][0], s[n][2 * h + 1][1]),
                             gqa_pack2<T>(s[n][2 * h + 1][2], s[n][2 * h + 1][3]));
        const int row = 32 * h + 4 * g + (c >> 2);  // (and 16 further on: the same swizzle)
        const uint8_t* base = vt + row * G::ROWB + (c & 1) * 8;
#pragma unroll
        for (int d = 0; d < OT; ++d) {
          const uint8_t* at = base + (((2 * d + ((c >> 1) & 1)) ^ G::swz_v(row)) << 4);
          struct {
            s16x4 a, b;
          } v{__builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)at),
              __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(at + 16 * G::ROWB))};
          const uint4 vf = __builtin_bit_cast(uint4, v);
#pragma unroll
          for (int n = 0; n < NT; ++n) o[n][d] = gqa_mma<T>(vf, pf[n], o[n][d]);
        }
      }
    }
  }
};

// A row's result: to `out`, or its piece's record in the workspace. o4: elements d .. d + 3.
template <typename T>
__device__ __forceinline__ void gqa_store(const GqaArgs& a, int tok, int head, int piece, bool direct, int d, f32x4 o4, float m,
                                          float l) {
  if (direct) {
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    T* dst = static_cast<T*>(a.out) + tok * a.o_st + head * a.o_sh + d;
    if (a.o_vec && d + 4 <= a.D) {
      store4<T>(dst, o4[0] * inv, o4[1] * inv, o4[2] * inv, o4[3] * inv);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (d + i < a.D) dst[i] = from_f32<T>(o4[i] * inv);
    }
    return;
  }
  const int64_t rec = ((int64_t)tok * a.Hkv * a.group + head) * a.pieces + piece;
  // (records of DW floats, a multiple of 4, so that a quad is one store)
  if (d < a.D) *reinterpret_cast<f32x4*>(a.ws + rec * a.DW + d) = o4;
  if (d == 0) *reinterpret_cast<float2*>(a.ws_ml + 2 * rec) = make_float2(m, l);
}

// Many rows: 4 wavefronts of 16 NT rows each share tiles of BN keys, in two LDS buffers.
template <typename T, int DP>
constexpr int gqa_bn() {
  return GqaType<T>::F32 ? (DP <= 64 ? 64 : DP <= 128 ? 32 : 16) : (DP <= 128 ? 64 : 32);
}

template <typename T, int DP, int NT, int BN, bool VEC>
__device__ __forceinline__ void gqa_rows_step(const GqaArgs& a, GqaRows<T, DP, NT>& rows, const uint8_t* __restrict__ cur,
                                              uint8_t* __restrict__ nxt, const uint8_t* kbase, const uint8_t* vbase, int64_t off,
                                              bool more, int j0, uint64_t okmask, int wave, int lane) {
  constexpr int TB = BN * GqaTile<T, DP>::ROWB;
  if (more) gqa_fill<T, DP, BN, 256, VEC>(nxt, nxt + TB, kbase, vbase, off, a.D, wave, lane);
  if (rows.sees_any(j0, BN)) rows.template step<BN>(a, cur, cur + TB, j0, okmask, lane);
}

template <typename T, int DP, int NT, bool VEC>
__global__ __launch_bounds__(256, DP <= 128 ? 2 : 1) void gqa_rows_kernel(const GqaArgs a) {
  constexpr int BN = gqa_bn<T, DP>(), TB = BN * GqaTile<T, DP>::ROWB;
  extern __shared__ __align__(1024) uint8_t smem[];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  int kvh, split;
  const GqaPlan p = gqa_block_plan(a, blockIdx.x, lane, kvh, split);
  if (split >= p.live || p.rows <= p.row0) return;
  GqaRows<T, DP, NT> rows;
  const int row0 = p.row0 + wave * 16 * NT;
  rows.init(a, p, row0, kvh, lane);
  const uint8_t* kbase = static_cast<const uint8_t*>(a.kp) + kvh * a.kv_sh * (int64_t)sizeof(T);
  const uint8_t* vbase = static_cast<const uint8_t*>(a.vp) + kvh * a.kv_sh * (int64_t)sizeof(T);
  const int t0 = split * p.per, t1 = min(p.tiles, t0 + p.per);
  // lane i looks up key i of a tile, two tiles ahead of its use
  auto key_in = [&](int t) { const int j = p.lo + t * BN + lane; return lane < BN && t < t1 && j >= p.klo && j < p.khi; };
  auto look = [&](int t) { return key_in(t) ? p.table[gqa_block_of(a, p.lo + t * BN + lane)] : -1; };
  if (t0 < t1) {
    int blk = look(t0);
    int64_t off = gqa_key_offset(a, p.lo + t0 * BN + lane, blk, key_in(t0), sizeof(T));
    uint64_t ok = __ballot(off >= 0);
    blk = look(t0 + 1);
    gqa_fill<T, DP, BN, 256, VEC>(smem, smem + TB, kbase, vbase, off, a.D, wave, lane);
    for (int t = t0; t < t1; ++t) {
      asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
      off = gqa_key_offset(a, p.lo + (t + 1) * BN + lane, blk, key_in(t + 1), sizeof(T));
      const uint64_t ok1 = __ballot(off >= 0);
      blk = look(t + 2);
      const int cur = ((t - t0) & 1) * 2 * TB;
      gqa_rows_step<T, DP, NT, BN, VEC>(a, rows, smem + cur, smem + (2 * TB - cur), kbase, vbase, off, t + 1 < t1,
                                        p.lo + t * BN, ok, wave, lane);
      ok = ok1;
    }
  }
  const int g = lane >> 4;
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    const int r = row0 + 16 * n + (lane & 15);
    const float l = gqa_row_sum(rows.l[n]);
    if (r < p.rows) {
      const int tok = p.tok0 + r / a.group, head = kvh * a.group + r % a.group;
#pragma unroll
      for (int d = 0; d < DP / 16; ++d)
        gqa_store<T>(a, tok, head, a.piece0 + split, p.direct, 16 * d + 4 * g, rows.o[n][d], rows.m[n], l);
    }
  }
}

// Few rows: the NW wavefronts of a block hold the same 16 NT rows and take WK keys each of a
// step of NW WK keys, each with LDS buffers of its own, so that no wavefront waits for another
// before the end, where their states are joined through LDS.
template <typename T, int DP>
constexpr int gqa_wk() { return GqaType<T>::F32 ? (DP <= 64 ? 32 : 16) : 32; }
template <typename T, int DP>
constexpr int gqa_nw() { return gqa_wk<T, DP>() * GqaTile<T, DP>::ROWB > 8192 ? 2 : 4; }

template <typename T, int DP, int NT, int WK>
__device__ __forceinline__ void gqa_keys_step(const GqaArgs& a, GqaRows<T, DP, NT>& rows, const uint8_t* __restrict__ cur,
                                              uint8_t* __restrict__ nxt, const uint8_t* kbase, const uint8_t* vbase, int64_t off,
                                              bool more, int j0, uint64_t okmask, int lane) {
  constexpr int TB = WK * GqaTile<T, DP>::ROWB;
  if (more) gqa_fill<T, DP, WK, 64, true>(nxt, nxt + TB, kbase, vbase, off, a.D, 0, lane);
  if (okmask != 0 && rows.sees_any(j0, WK)) rows.template step<WK>(a, cur, cur + TB, j0, okmask, lane);
}

template <typename T, int DP, int NT>
__global__ __launch_bounds__(256, 1) void gqa_keys_kernel(const GqaArgs a) {
  constexpr int WK = gqa_wk<T, DP>(), NW = gqa_nw<T, DP>(), TB = WK * GqaTile<T, DP>::ROWB, BN = NW * WK;
  constexpr int OL = DP + 4;  // floats of an output row in LDS
  extern __shared__ __align__(1024) uint8_t smem[];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  int kvh, split;
  const GqaPlan p = gqa_block_plan(a, blockIdx.x, lane, kvh, split);
  if (split >= p.live || p.rows <= p.row0) return;
  GqaRows<T, DP, NT> rows;
  rows.init(a, p, p.row0, kvh, lane);
  const uint8_t* kbase = static_cast<const uint8_t*>(a.kp) + kvh * a.kv_sh * (int64_t)sizeof(T);
  const uint8_t* vbase = static_cast<const uint8_t*>(a.vp) + kvh * a.kv_sh * (int64_t)sizeof(T);
  const int t0 = split * p.per, t1 = min(p.tiles, t0 + p.per);
  uint8_t* mine = smem + wave * 4 * TB;
  auto first = [&](int t) { return p.lo + t * BN + wave * WK; };
  auto key_in = [&](int t) { const int j = first(t) + lane; return lane < WK && t < t1 && j >= p.klo && j < p.khi; };
  auto look = [&](int t) { return key_in(t) ? p.table[gqa_block_of(a, first(t) + lane)] : -1; };
  if (t0 < t1) {
    int blk = look(t0);
    int64_t off = gqa_key_offset(a, first(t0) + lane, blk, key_in(t0), sizeof(T));
    uint64_t ok = __ballot(off >= 0);
    blk = look(t0 + 1);
    gqa_fill<T, DP, WK, 64, true>(mine, mine + TB, kbase, vbase, off, a.D, 0, lane);
    for (int t = t0; t < t1; ++t) {
      asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
      off = gqa_key_offset(a, first(t + 1) + lane, blk, key_in(t + 1), sizeof(T));
      const uint64_t ok1 = __ballot(off >= 0);
      blk = look(t + 2);
      const int cur = ((t - t0) & 1) * 2 * TB;
      gqa_keys_step<T, DP, NT, WK>(a, rows, mine + cur, mine + (2 * TB - cur), kbase, vbase, off, t + 1 < t1, first(t), ok, lane);
      ok = ok1;
    }
  }
  // join the wavefronts' states
  float* ol = reinterpret_cast<float*>(smem);                // [NW][16 NT][OL]
  float* ml = ol + NW * 16 * NT * OL;                        // [NW][16 NT][2]
  __syncthreads();
  const int g = lane >> 4;
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    const int r = 16 * n + (lane & 15);
    const float l = gqa_row_sum(rows.l[n]);
#pragma unroll
    for (int d = 0; d < DP / 16; ++d)
      *reinterpret_cast<f32x4*>(ol + (wave * 16 * NT + r) * OL + 16 * d + 4 * g) = rows.o[n][d];
    if (g == 0) *reinterpret_cast<float2*>(ml + (wave * 16 * NT + r) * 2) = make_float2(rows.m[n], l);
  }
  __syncthreads();
  for (int e = threadIdx.x; e < 16 * NT * (DP / 4); e += NW * 64) {
    const int rr = e / (DP / 4), d = (e % (DP / 4)) * 4, r = p.row0 + rr;
    if (r >= p.rows || d >= a.D) continue;
    float M = -3.402823466e38f, L = 0.0f;
    float2 x[NW];
#pragma unroll
    for (int w = 0; w < NW; ++w) {
      x[w] = *reinterpret_cast<const float2*>(ml + (w * 16 * NT + rr) * 2);
      M = fmaxf(M, x[w].x);
    }
    f32x4 acc{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < NW; ++w) {
      const float f = __builtin_amdgcn_exp2f(x[w].x - M);
      L += x[w].y * f;
      acc += *reinterpret_cast<const f32x4*>(ol + (w * 16 * NT + rr) * OL + d) * f;
    }
    const int tok = p.tok0 + r / a.group, head = kvh * a.group + r % a.group;
    gqa_store<T>(a, tok, head, a.piece0 + split, p.direct, d, acc, M, L);
  }
}

template <typename T, int DP, int NT>
constexpr int gqa_keys_lds() {
  constexpr int NW = gqa_nw<T, DP>();
  constexpr int tiles = NW * 4 * gqa_wk<T, DP>() * GqaTile<T, DP>::ROWB, join = NW * 16 * NT * (DP + 4 + 2) * 4;
  return tiles > join ? tiles : join;
}

// Launches KERN with `lds` bytes of dynamic LDS, whose limit is raised once a function and device.
template <void (*KERN)(const GqaArgs)>
int gqa_launch_kernel(const GqaArgs& a, int64_t blocks, int threads, int lds, hipStream_t st) {
  static std::atomic<uint64_t> raised{0};
  int dev = 0;
  if (lds > 64 * 1024 && hipGetDevice(&dev) == hipSuccess && !(raised.load() >> (dev & 63) & 1)) {
    if (hipFuncSetAttribute((const void*)KERN, hipFuncAttributeMaxDynamicSharedMemorySize, lds) != hipSuccess)
      return fail(MLS_ERR_HIP, "paged attention: cannot reserve %d bytes of LDS", lds);
    raised.fetch_or(1ull << (dev & 63));
  }
  hipLaunchKernelGGL(KERN, dim3((unsigned)blocks), dim3(threads), lds, st, a);
  return check_launch("paged attention");
}

template <typename T, int DP>
int gqa_launch_dp(const GqaArgs& a, const GqaShape& s, int64_t blocks, hipStream_t st) {
  if (s.keys) {
    constexpr int threads = gqa_nw<T, DP>() * 64, l1 = gqa_keys_lds<T, DP, 1>(), l2 = gqa_keys_lds<T, DP, 2>();
    if (s.nt == 1) return gqa_launch_kernel<gqa_keys_kernel<T, DP, 1>>(a, blocks, threads, l1, st);
    return gqa_launch_kernel<gqa_keys_kernel<T, DP, 2>>(a, blocks, threads, l2, st);
  }
  constexpr int lds = 4 * gqa_bn<T, DP>() * GqaTile<T, DP>::ROWB;
  if (!s.vec) return gqa_launch_kernel<gqa_rows_kernel<T, DP, 1, false>>(a, blocks, 256, lds, st);
  if (s.nt == 1) return gqa_launch_kernel<gqa_rows_kernel<T, DP, 1, true>>(a, blocks, 256, lds, st);
  return gqa_launch_kernel<gqa_rows_kernel<T, DP, 2, true>>(a, blocks, 256, lds, st);
}

template <typename T, int DP>
void gqa_tiles_dp(GqaShape& s) {
  s.bn = s.keys ? gqa_nw<T, DP>() * gqa_wk<T, DP>() : gqa_bn<T, DP>();
}

template <typename T>
int gqa_launch(const GqaArgs& a, const GqaShape& s, int64_t blocks, hipStream_t st) {
  switch (s.dp) {
    case 64: return gqa_launch_dp<T, 64>(a, s, blocks, st);
    case 96: return gqa_launch_dp<T, 96>(a, s, blocks, st);
    case 128: return gqa_launch_dp<T, 128>(a, s, blocks, st);
    default: return gqa_launch_dp<T, 256>(a, s, blocks, st);
  }
}

template <typename T>
void gqa_tiles(GqaShape& s) {
  switch (s.dp) {
    case 64: return gqa_tiles_dp<T, 64>(s);
    case 96: return gqa_tiles_dp<T, 96>(s);
    case 128: return gqa_tiles_dp<T, 128>(s);
    default: return gqa_tiles_dp<T, 256>(s);
  }
}

}  // namespace mls
