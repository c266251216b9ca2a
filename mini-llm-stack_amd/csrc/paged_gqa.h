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

typedef float f32x2 __attribute__((ext_vector_type(2)));

// Two values rounded to T, one instruction (round to nearest even).
template <typename T>
__device__ __forceinline__ uint32_t gqa_pack2(float lo, float hi) {
  const f32x2 v{lo, hi};
  if constexpr (__is_same(T, __bf16)) return __builtin_bit_cast(uint32_t, __builtin_convertvector(v, bf16x2));
  else return __builtin_bit_cast(uint32_t, __builtin_convertvector(v, f16x2));
}
// What the rounding left: (lo, hi) less the two values in `p`.
template <typename T>
__device__ __forceinline__ uint32_t gqa_rest2(float lo, float hi, uint32_t p) {
  if constexpr (__is_same(T, __bf16)) {
    return gqa_pack2<T>(lo - __uint_as_float(p << 16), hi - __uint_as_float(p & 0xFFFF0000u));
  } else {
    const f16x2 h = __builtin_bit_cast(f16x2, p);
    return gqa_pack2<T>(lo - (float)h.x, hi - (float)h.y);
  }
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

// Loads the K rows (V = false) or V rows of BN keys into LDS, by WAVES wavefronts, of which this is
// `wave`. off: lane i's is key i's byte offset in the pool, -1 for a key to be read as zeros. `whole`
// (uniform): no such key, no padded elements, and an instruction's rows all lie in one cache block, so
// that they need one address, in scalar registers. (With an address a row for every lane, the loads'
// addresses alone are 78 vector instructions a tile of 64 keys, a third of the main loop's.)
template <typename T, int DP, int BN, int WAVES, bool VEC, bool V>
__device__ __forceinline__ void gqa_fill(const GqaArgs& a, uint8_t* dst, const uint8_t* base, int64_t off, bool whole, int wave,
                                         int lane) {
  using G = GqaTile<T, DP>;
  constexpr int ROWS = 64 / G::CPR, ITER = BN / ROWS / WAVES;  // rows of one instruction; instructions
  static_assert(BN <= 64 && ITER * ROWS * WAVES == BN, "whole instructions");
  const int r = lane / G::CPR, c = lane % G::CPR;
  if (VEC && whole) {
#pragma unroll
    for (int u = 0; u < ITER; ++u) {
      const int row = (u * WAVES + wave) * ROWS;  // (uniform)
      const int64_t o = ((int64_t)__builtin_amdgcn_readlane((int)(off >> 32), row) << 32) |
                        (uint32_t)__builtin_amdgcn_readlane((int)off, row);
      const int cc = c ^ (V ? G::swz_v(row + r) : G::swz_k(row + r));
      const uint32_t in = (uint32_t)r * (uint32_t)a.kv_st * (uint32_t)sizeof(T) + cc * 16;
      gqa_lds_load16(base + o + in, dst + (u * WAVES + wave) * 1024);
    }
    return;
  }
#pragma unroll
  for (int u = 0; u < ITER; ++u) {
    const int row = (u * WAVES + wave) * ROWS + r;
    const int lo = __shfl((int)off, row, 64), hi = __shfl((int)(off >> 32), row, 64);
    const int64_t o = ((int64_t)hi << 32) | (uint32_t)lo;
    const int cc = c ^ (V ? G::swz_v(row) : G::swz_k(row));
    uint8_t* d = dst + (u * WAVES + wave) * 1024;
    if constexpr (VEC) {
      const uint8_t* zero = reinterpret_cast<const uint8_t*>(gqa_zeros);
      gqa_lds_load16(hi >= 0 && cc * G::CE < a.D ? base + o + cc * 16 : zero, d);
    } else {
      T x[G::CE];
#pragma unroll
      for (int e = 0; e < G::CE; ++e) {
        const int dd = cc * G::CE + e;
        x[e] = hi >= 0 && dd < a.D ? reinterpret_cast<const T*>(base + o)[dd] : (T)0.0f;
      }
      *reinterpret_cast<uint4*>(d + lane * 16) = __builtin_bit_cast(uint4, x);
    }
  }
}

// The place of key `key` in the pools (bytes from a head's base), from its block id.
__device__ __forceinline__ int64_t gqa_key_offset(const GqaArgs& a, int key, int blk, bool in, int esz) {
  const bool ok = in && blk >= 0 && blk < a.num_blocks;
  const int t = key - gqa_block_of(a, key) * a.BS;
  return ok ? ((int64_t)blk * a.kv_sb + (int64_t)t * a.kv_st) * esz : -1;
}

// One wavefront's rows: 16 NT query rows with their softmax state. SPLIT: P as two parts of the
// inputs' type (where loads, not products, bound the kernel), else rounded once.
template <typename T, int DP, int NT, bool SPLIT>
struct GqaRows {
  using G = GqaTile<T, DP>;
  using K = GqaType<T>;
  static constexpr int QT = DP / (4 * K::CE), OT = DP / 16;
  // 16-bit: the sum of a row's weights is a product with ones, so it costs no vector
  // instructions, and counts the weights as rounded; every lane of the row holds it. fp32: lanes' parts.
  static constexpr bool LMMA = !K::F32;
  uint4 q[NT][QT];
  f32x4 o[NT][OT], ol[NT];
  float m[NT];
  int lo[NT], hi[NT], pos[NT];  // the keys that a row sees: [lo, hi)
  float slope[NT];              // times log2(e)
  int lo_min, lo_max, hi_min, hi_max;  // over the wavefront's rows

  // row0: the wavefront's first packed row of the tile's sequence
  __device__ __forceinline__ void init(const GqaArgs& a, const GqaPlan& p, int row0, int kvh, int lane) {
    const int g = lane >> 4;
    gqa_wave_range(a, p, row0, min(row0 + 16 * NT, p.rows) - 1, lane, lo_min, lo_max, hi_min, hi_max);
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      m[n] = -3.402823466e38f;
      ol[n] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int d = 0; d < OT; ++d) o[n][d] = f32x4{0.f, 0.f, 0.f, 0.f};
      const int r = row0 + 16 * n + (lane & 15);
      const bool in = r < p.rows;
      const int t = r / a.group, tok = min(p.tok0 + t, a.T - 1), head = kvh * a.group + r - t * a.group;
      gqa_row_range(a, p, tok, lo[n], hi[n], pos[n]);
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
  }

  // Whether every row of the wavefront sees all of the keys [j, j + n), and whether any row sees any
  __device__ __forceinline__ bool sees_all(int j, int n) const { return lo_max <= j && j + n <= hi_min; }
  __device__ __forceinline__ bool sees_any(int j, int n) const { return lo_min < j + n && j < hi_max; }

  // S = K Q^T for the BN keys in kt; a sub-tile's fragments are read while the one before it multiplies
  template <int BN>
  __device__ __forceinline__ void scores(const uint8_t* kt, int lane, f32x4 (&s)[NT][BN / 16]) const {
    constexpr int KT = BN / 16;
    const int g = lane >> 4, c = lane & 15;
    const uint8_t* at[QT];
#pragma unroll
    for (int t = 0; t < QT; ++t) at[t] = kt + c * G::ROWB + (((4 * t + g) ^ G::swz_k(c)) << 4);
    uint4 kf[2][QT];
#pragma unroll
    for (int t = 0; t < QT; ++t) kf[0][t] = *reinterpret_cast<const uint4*>(at[t]);
#pragma unroll
    for (int k = 0; k < KT; ++k) {
      if (k + 1 < KT)
#pragma unroll
        for (int t = 0; t < QT; ++t) kf[(k + 1) & 1][t] = *reinterpret_cast<const uint4*>(at[t] + (k + 1) * 16 * G::ROWB);
#pragma unroll
      for (int n = 0; n < NT; ++n) s[n][k] = gqa_mma<T>(kf[k & 1][0], q[n][0], f32x4{0.f, 0.f, 0.f, 0.f});
#pragma unroll
      for (int t = 1; t < QT; ++t)
#pragma unroll
        for (int n = 0; n < NT; ++n) s[n][k] = gqa_mma<T>(kf[k & 1][t], q[n][t], s[n][k]);
    }
  }

  // Scores -> weights (s becomes P), with the row's state rescaled where its reference moves. okmask: the
  // keys of [j0, j0 + BN) that are there at all.
  template <int BN>
  __device__ __forceinline__ void weigh(const GqaArgs& a, f32x4 (&s)[NT][BN / 16], int j0, uint64_t okmask, int lane) {
    constexpr int KT = BN / 16;
    const int g = lane >> 4;
    // scores in log2 units: s * cc
    float cc = a.c;
    if (!a.simple) {
      cc = 1.0f;
      scored<KT>(a, s, j0, g);
    }
    constexpr uint64_t FULL = BN == 64 ? ~0ull : (1ull << (BN & 63)) - 1;
    if (okmask != FULL || !sees_all(j0, BN)) {
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
    if (__builtin_expect(__any(over), 0)) {
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        const float mn = fmaxf(m[n], gqa_row_max(mx[n]) - K::OFF);
        const float f = __builtin_amdgcn_exp2f(m[n] - mn);
        m[n] = mn;
        ol[n] *= f;
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
          if constexpr (!LMMA) ol[n][0] += s[n][k][i];
        }
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

  // O^T += V^T P^T, and the weights' sums
  template <int BN>
  __device__ __forceinline__ void product(const f32x4 (&s)[NT][BN / 16], const uint8_t* vt, int lane) {
    const int g = lane >> 4, c = lane & 15;
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
      constexpr uint32_t ONE = __is_same(T, __bf16) ? 0x3F803F80u : 0x3C003C00u;
      const uint4 ones = make_uint4(ONE, ONE, ONE, ONE);
      const int row = 4 * g + (c >> 2);  // (and 16, 32 further on: the same swizzle)
      const uint8_t* at[OT];
#pragma unroll
      for (int d = 0; d < OT; ++d)
        at[d] = vt + row * G::ROWB + (c & 1) * 8 + (((2 * d + ((c >> 1) & 1)) ^ G::swz_v(row)) << 4);
#pragma unroll
      for (int h = 0; h < BN / 32; ++h) {
        uint4 pf[NT], pr[NT];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          const f32x4 x = s[n][2 * h], y = s[n][2 * h + 1];
          pf[n] = make_uint4(gqa_pack2<T>(x[0], x[1]), gqa_pack2<T>(x[2], x[3]), gqa_pack2<T>(y[0], y[1]), gqa_pack2<T>(y[2], y[3]));
          if constexpr (SPLIT)
            pr[n] = make_uint4(gqa_rest2<T>(x[0], x[1], pf[n].x), gqa_rest2<T>(x[2], x[3], pf[n].y),
                               gqa_rest2<T>(y[0], y[1], pf[n].z), gqa_rest2<T>(y[2], y[3], pf[n].w));
        }
#pragma unroll
        for (int d = 0; d < OT; ++d) {
          const uint8_t* p = at[d] + h * 32 * G::ROWB;
          struct {
            s16x4 a, b;
          } v{__builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)p),
              __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(p + 16 * G::ROWB))};
          const uint4 vf = __builtin_bit_cast(uint4, v);
#pragma unroll
          for (int n = 0; n < NT; ++n) o[n][d] = gqa_mma<T>(vf, pf[n], o[n][d]);
          if constexpr (SPLIT)
#pragma unroll
            for (int n = 0; n < NT; ++n) o[n][d] = gqa_mma<T>(vf, pr[n], o[n][d]);
        }
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          ol[n] = gqa_mma<T>(ones, pf[n], ol[n]);
          if constexpr (SPLIT) ol[n] = gqa_mma<T>(ones, pr[n], ol[n]);
        }
      }
    }
  }

  __device__ __forceinline__ float sum_of(int n) const { return LMMA ? ol[n][0] : gqa_row_sum(ol[n][0]); }
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

// How many pieces a row has, for the join; written by its first.
__device__ __forceinline__ void gqa_store_live(const GqaArgs& a, int tok, int head, int split, int live) {
  if (split == 0 && a.ws_live) a.ws_live[(int64_t)tok * a.Hkv * a.group + head] = live;
}

// Many rows: 4 wavefronts of 16 NT rows each share tiles of BN keys, in two LDS buffers.
template <typename T, int DP>
constexpr int gqa_bn() {
  return GqaType<T>::F32 ? (DP <= 64 ? 64 : DP <= 128 ? 32 : 16) : (DP <= 128 ? 64 : 32);
}

template <typename T, int DP, int NT, int BN, bool VEC>
__device__ __forceinline__ void gqa_rows_step(const GqaArgs& a, GqaRows<T, DP, NT, false>& rows, const uint8_t* __restrict__ cur,
                                              uint8_t* __restrict__ nxt, const uint8_t* kbase, const uint8_t* vbase, int64_t off,
                                              bool more, bool whole, int j0, uint64_t okmask, int wave, int lane) {
  constexpr int TB = BN * GqaTile<T, DP>::ROWB;
  if (more) {
    gqa_fill<T, DP, BN, 4, VEC, false>(a, nxt, kbase, off, whole, wave, lane);
    gqa_fill<T, DP, BN, 4, VEC, true>(a, nxt + TB, vbase, off, whole, wave, lane);
  }
  if (!rows.sees_any(j0, BN)) return;
  f32x4 s[NT][BN / 16];
  rows.template scores<BN>(cur, lane, s);
  rows.template weigh<BN>(a, s, j0, okmask, lane);
  rows.template product<BN>(s, cur + TB, lane);
}

template <typename T, int DP, int NT, bool VEC>
__global__ __launch_bounds__(256, DP <= 128 ? 2 : 1) void gqa_rows_kernel(const GqaArgs a) {
  constexpr int BN = gqa_bn<T, DP>(), TB = BN * GqaTile<T, DP>::ROWB;
  constexpr uint64_t FULL = BN == 64 ? ~0ull : (1ull << (BN & 63)) - 1;
  extern __shared__ __align__(1024) uint8_t smem[];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  int kvh, split;
  const GqaPlan p = gqa_block_plan(a, blockIdx.x, lane, kvh, split);
  if (split >= p.live || p.rows <= p.row0) return;
  GqaRows<T, DP, NT, false> rows;
  const int row0 = p.row0 + wave * 16 * NT;
  rows.init(a, p, row0, kvh, lane);
  const uint8_t* kbase = static_cast<const uint8_t*>(a.kp) + kvh * a.kv_sh * (int64_t)sizeof(T);
  const uint8_t* vbase = static_cast<const uint8_t*>(a.vp) + kvh * a.kv_sh * (int64_t)sizeof(T);
  const bool blocks = a.D == GqaTile<T, DP>::DL && a.BS % (64 / GqaTile<T, DP>::CPR) == 0 && a.kv_st < (1 << 24);
  const int t0 = split * p.per, t1 = min(p.tiles, t0 + p.per);
  // lane i looks up key i of a tile, two tiles ahead of its use
  auto key_in = [&](int t) { const int j = p.lo + t * BN + lane; return lane < BN && t < t1 && j >= p.klo && j < p.khi; };
  auto look = [&](int t) { return key_in(t) ? p.table[gqa_block_of(a, p.lo + t * BN + lane)] : -1; };
  if (t0 < t1) {
    int blk = look(t0);
    int64_t off = gqa_key_offset(a, p.lo + t0 * BN + lane, blk, key_in(t0), sizeof(T));
    uint64_t ok = __ballot(off >= 0);
    blk = look(t0 + 1);
    gqa_fill<T, DP, BN, 4, VEC, false>(a, smem, kbase, off, blocks && ok == FULL, wave, lane);
    gqa_fill<T, DP, BN, 4, VEC, true>(a, smem + TB, vbase, off, blocks && ok == FULL, wave, lane);
    auto step = [&](int t, const uint8_t* cur, uint8_t* nxt) __attribute__((always_inline)) {
      asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
      off = gqa_key_offset(a, p.lo + (t + 1) * BN + lane, blk, key_in(t + 1), sizeof(T));
      const uint64_t ok1 = __ballot(off >= 0);
      blk = look(t + 2);
      gqa_rows_step<T, DP, NT, BN, VEC>(a, rows, cur, nxt, kbase, vbase, off, t + 1 < t1, blocks && ok1 == FULL, p.lo + t * BN, ok,
                                        wave, lane);
      ok = ok1;
    };
    for (int t = t0; t < t1; t += 2) {  // (in pairs: LDS addresses are constants then)
      step(t, smem, smem + 2 * TB);
      if (t + 1 < t1) step(t + 1, smem + 2 * TB, smem);
    }
  }
  const int g = lane >> 4;
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    const int r = row0 + 16 * n + (lane & 15);
    const float l = rows.sum_of(n);
    if (r < p.rows) {
      const int tok = p.tok0 + r / a.group, head = kvh * a.group + r % a.group;
#pragma unroll
      for (int d = 0; d < DP / 16; ++d)
        gqa_store<T>(a, tok, head, a.piece0 + split, p.direct, 16 * d + 4 * g, rows.o[n][d], rows.m[n], l);
      if (g == 0) gqa_store_live(a, tok, head, split, p.live);
    }
  }
}

// Few rows: the NW wavefronts of a block hold the same 16 NT rows and take WK keys each of a
// step of NW WK keys, each with LDS of its own, so that no wavefront waits for another before the end,
// where their states are joined through LDS. A wavefront has one K and one V buffer: the next K
// tile is on its way from the moment this one's scores are done, the next V tile from the end of
// this one's product, so that 8 wavefronts a CU (64 KB of LDS a block) keep 64 to 128 KB of loads in
// flight. (With two buffers of each and 4 wavefronts a CU, 64 KB in flight at most: 40
// sequences of 1 to 4096 tokens, 32 heads of 128 over 8 K/V heads, 45 us.)
template <typename T, int DP>
constexpr int gqa_wk() { return GqaType<T>::F32 ? (DP <= 64 ? 32 : 16) : 32; }
template <typename T, int DP>
constexpr int gqa_nw() { return gqa_wk<T, DP>() * GqaTile<T, DP>::ROWB > 8192 ? 2 : 4; }

template <typename T, int DP, int NT, int WK>
__device__ __forceinline__ void gqa_keys_step(const GqaArgs& a, GqaRows<T, DP, NT, !GqaType<T>::F32>& rows, uint8_t* __restrict__ kt,
                                              uint8_t* __restrict__ vt, const uint8_t* kbase, const uint8_t* vbase, int64_t off,
                                              bool more, bool whole, int j0, uint64_t okmask, int lane) {
  constexpr int PER = WK * GqaTile<T, DP>::ROWB / 1024;  // loads of a K or V tile
  f32x4 s[NT][WK / 16];
  // loads complete in order, and this K tile's are older than the V tile's (a table entry may follow those)
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(PER) : "memory");
  rows.template scores<WK>(kt, lane, s);
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // (K is read)
  if (more) gqa_fill<T, DP, WK, 1, true, false>(a, kt, kbase, off, whole, 0, lane);
  rows.template weigh<WK>(a, s, j0, okmask, lane);
  if (more) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(PER) : "memory");
  else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  rows.template product<WK>(s, vt, lane);
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // (V is read)
  if (more) gqa_fill<T, DP, WK, 1, true, true>(a, vt, vbase, off, whole, 0, lane);
}

template <typename T, int DP, int NT>
__global__ __launch_bounds__((gqa_nw<T, DP>() * 64), (gqa_nw<T, DP>() / 2)) void gqa_keys_kernel(const GqaArgs a) {
  constexpr int WK = gqa_wk<T, DP>(), NW = gqa_nw<T, DP>(), TB = WK * GqaTile<T, DP>::ROWB, BN = NW * WK;
  constexpr uint64_t FULL = (1ull << WK) - 1;
  constexpr int OL = DP + 4;  // floats of an output row in LDS
  extern __shared__ __align__(1024) uint8_t smem[];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  int kvh, split;
  const GqaPlan p = gqa_block_plan(a, blockIdx.x, lane, kvh, split);
  if (split >= p.live || p.rows <= p.row0) return;
  GqaRows<T, DP, NT, !GqaType<T>::F32> rows;
  const uint8_t* kbase = static_cast<const uint8_t*>(a.kp) + kvh * a.kv_sh * (int64_t)sizeof(T);
  const uint8_t* vbase = static_cast<const uint8_t*>(a.vp) + kvh * a.kv_sh * (int64_t)sizeof(T);
  const bool blocks = a.D == GqaTile<T, DP>::DL && a.BS % (64 / GqaTile<T, DP>::CPR) == 0 && a.kv_st < (1 << 24);
  int t0 = split * p.per, t1 = min(p.tiles, t0 + p.per);
  // this wavefront's first and last steps may hold none of its keys
  if (p.lo + t0 * BN + (wave + 1) * WK <= p.klo) ++t0;
  t1 = min(t1, (p.khi - p.lo - wave * WK + BN - 1) / BN);
  uint8_t *kt = smem + wave * 2 * TB, *vt = kt + TB;
  auto first = [&](int t) { return p.lo + t * BN + wave * WK; };
  auto key_in = [&](int t) { const int j = first(t) + lane; return lane < WK && t < t1 && j >= p.klo && j < p.khi; };
  auto look = [&](int t) { return key_in(t) ? p.table[gqa_block_of(a, first(t) + lane)] : -1; };
  int64_t off = -1;
  uint64_t ok = 0;
  int blk = -1;
  if (t0 < t1) {
    blk = look(t0);
    off = gqa_key_offset(a, first(t0) + lane, blk, key_in(t0), sizeof(T));
    ok = __ballot(off >= 0);
    gqa_fill<T, DP, WK, 1, true, false>(a, kt, kbase, off, blocks && ok == FULL, 0, lane);
    gqa_fill<T, DP, WK, 1, true, true>(a, vt, vbase, off, blocks && ok == FULL, 0, lane);
  }
  rows.init(a, p, p.row0, kvh, lane);
  blk = t0 + 1 < t1 ? look(t0 + 1) : -1;
  for (int t = t0; t < t1; ++t) {
    off = gqa_key_offset(a, first(t + 1) + lane, blk, key_in(t + 1), sizeof(T));
    const uint64_t ok1 = __ballot(off >= 0);
    blk = look(t + 2);
    gqa_keys_step<T, DP, NT, WK>(a, rows, kt, vt, kbase, vbase, off, t + 1 < t1, blocks && ok1 == FULL, first(t), ok, lane);
    ok = ok1;
  }
  // join the wavefronts' states
  float* ol = reinterpret_cast<float*>(smem);                // [NW][16 NT][OL]
  float* ml = ol + NW * 16 * NT * OL;                        // [NW][16 NT][2]
  __syncthreads();
  const int g = lane >> 4;
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    const int r = 16 * n + (lane & 15);
    const float l = rows.sum_of(n);
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
    if (d == 0) gqa_store_live(a, tok, head, split, p.live);
  }
}

template <typename T, int DP, int NT>
constexpr int gqa_keys_lds() {
  constexpr int NW = gqa_nw<T, DP>();
  constexpr int tiles = NW * 2 * gqa_wk<T, DP>() * GqaTile<T, DP>::ROWB, join = NW * 16 * NT * (DP + 4 + 2) * 4;
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
