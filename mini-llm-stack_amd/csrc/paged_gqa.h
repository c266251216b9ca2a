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
// rescales l and O. All statistics are fp32. For the product with V, P is rounded to the inputs' type (half a
// step of each weight; l sums the weights as rounded, so that a row's shares still add to 1), but in the kernel over
// keys, whose matrix unit has room: there P is two parts of that type.
#pragma once

#include <atomic>

#include "common.h"
#include "paged_gqa_args.h"

namespace mls {

typedef short s16x4 __attribute__((ext_vector_type(4)));

// Zeros: what a lane loads for a key outside its range, of a block id outside the pool, or for
// elements past the head dim. A whole row of the widest head.
static __device__ __align__(16) const uint32_t gqa_zeros[256] = {};

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
// Chunk c of K row r sits at c ^ (r & 15) (16 lanes read one chunk of 16 rows at once); of V row r at c ^ 2 (r & 7) (16-bit: the four rows that
// one group of 16 lanes reads transposed, 32 bytes of each, lie in different banks) or, fp32,
// c ^ 4 ((r >> 2) & 3) (four lane groups read 64 bytes of rows 4 apart).
template <typename T, int DP>
struct GqaTile {
  static constexpr int CE = GqaType<T>::CE;
  static constexpr int DL = DP <= 64 ? 64 : DP <= 128 ? 128 : 256;
  static constexpr int CPR = DL / CE, ROWB = DL * (int)sizeof(T);
  __device__ static __forceinline__ int swz_k(int r) { return r & (CPR >= 16 ? 15 : 7); }
  __device__ static __forceinline__ int swz_v(int r) {
    if constexpr (GqaType<T>::F32) return ((r >> 2) & 3) << 2;
    return (r << 1) & (CPR >= 16 ? 14 : 6);
  }
};

// A value that the compiler takes as new here: what rarely taken branches make of it is not made
// ahead of the loop around them, in registers that the loop then lacks.
__device__ __forceinline__ int gqa_here(int v) {
  asm volatile("" : "+v"(v));
  return v;
}

// Before a main loop: the loads so far (q, block ids) have landed, said in a way that the compiler
// counts; else their first use in the loop would wait, in every pass, for the loop's loads.
__device__ __forceinline__ void gqa_landed() { __builtin_amdgcn_s_waitcnt(0 | 0x70 | 0xF00); }

// A sequence's block ids: 128 of them in two registers, a lane each, so that a tile's lookup is no
// load (one that the counter of the tiles' own loads would make wait for those).
struct GqaTable {
  int tab, next, base;  // entries [base, base + 64) and [base + 64, base + 128)
  bool holes;           // an id of these that the tile may use is outside the pool
  __device__ __forceinline__ int load(const GqaArgs& a, const GqaPlan& p, int from, int lane) {
    const int e = from + lane;
    const bool in = p.khi > 0 && e <= gqa_block_of(a, p.khi - 1);
    const int blk = in ? p.table[e] : -1;
    holes = holes || __any(in && (blk < 0 || blk >= a.num_blocks));
    return blk < a.num_blocks ? blk : -1;
  }
  __device__ __forceinline__ void start(const GqaArgs& a, const GqaPlan& p, int j0, int lane) {
    holes = false;
    base = gqa_block_of(a, j0);
    tab = load(a, p, base, lane);
    next = load(a, p, base + 64, lane);
  }
  // Moves on to the tile from key j0 on (tiles in rising order).
  __device__ __forceinline__ void advance(const GqaArgs& a, const GqaPlan& p, int j0, int lane) {
    if (j0 >= p.khi) return;
    const int first = gqa_block_of(a, j0);
    while (first - base >= 64) {
      tab = next;
      base += 64;
      next = load(a, p, base + 64, lane);
      gqa_landed();  // (once in 64 blocks)
    }
  }
  // Lane i: the block of the tile's key j0 + i, negative for none. Called with all lanes on: ids come from
  // other lanes' registers, and a lane that is off gives 0, a block of the pool.
  __device__ __forceinline__ int block(const GqaArgs& a, int j0, int lane) const {
    const int i = gqa_block_of(a, j0 + lane) - base;
    const int x = __shfl(tab, i & 63, 64), y = __shfl(next, i & 63, 64);
    return i < 64 ? x : y;
  }
  // The same for one key, uniform
  __device__ __forceinline__ int block_at(const GqaArgs& a, int key) const {
    const int i = gqa_block_of(a, key) - base;
    const int x = __builtin_amdgcn_readlane(tab, i & 63), y = __builtin_amdgcn_readlane(next, i & 63);
    return i < 64 ? x : y;
  }
  // The keys of the tile that any row sees
  template <int N>
  __device__ __forceinline__ uint64_t seen(const GqaArgs& a, const GqaPlan& p, int j0, int lane) const {
    if (j0 >= p.klo && j0 + N <= p.khi && !holes) return N == 64 ? ~0ull : (1ull << (N & 63)) - 1;
    if (j0 >= p.khi) return 0;
    const int here = gqa_here(lane), key = j0 + here;
    const int blk = block(a, j0, here);  // (not within the condition, which switches lanes off)
    return __ballot(here < N && key >= p.klo && key < p.khi && blk >= 0);
  }
};

// 16 bytes of T: whether a value is an infinity or NaN; the values with zeros for those; a bit for each NaN
template <typename T>
__device__ __forceinline__ bool gqa_odd(T x) { return !(to_f32(x) * 0.0f == 0.0f); }
template <typename T>
__device__ __forceinline__ bool gqa_odd_chunk(const uint4& v) {
  const T* x = reinterpret_cast<const T*>(&v);
  bool odd = false;
#pragma unroll
  for (int e = 0; e < GqaType<T>::CE; ++e) odd = odd || gqa_odd<T>(x[e]);
  return odd;
}
template <typename T>
__device__ __forceinline__ uint4 gqa_finite(uint4 v) {
  T* x = reinterpret_cast<T*>(&v);
#pragma unroll
  for (int e = 0; e < GqaType<T>::CE; ++e) x[e] = gqa_odd<T>(x[e]) ? (T)0.0f : x[e];
  return v;
}
template <typename T>
__device__ __forceinline__ uint32_t gqa_nans(const uint4& v) {
  const T* x = reinterpret_cast<const T*>(&v);
  uint32_t b = 0;
#pragma unroll
  for (int e = 0; e < GqaType<T>::CE; ++e) b |= (to_f32(x[e]) != to_f32(x[e]) ? 1u : 0u) << e;
  return b;
}

// Elements [d, d + CE) of a row of D, zeros past its end
template <typename T>
__device__ __forceinline__ uint4 gqa_chunk(const GqaArgs& a, const T* row, int d) {
  uint4 v = make_uint4(0, 0, 0, 0);
  if (a.kv_vec) {
    if (d < a.D) v = *reinterpret_cast<const uint4*>(row + d);
  } else {
    T x[GqaType<T>::CE];
#pragma unroll
    for (int e = 0; e < GqaType<T>::CE; ++e) x[e] = d + e < a.D ? row[d + e] : (T)0.0f;
    v = __builtin_bit_cast(uint4, x);
  }
  return v;
}

// Loads of a tile of BN keys by WAVES wavefronts: rows of one instruction, instructions of one wavefront.
template <typename T, int DP, int BN, int WAVES>
struct GqaFill {
  using G = GqaTile<T, DP>;
  static constexpr int ROWS = 64 / G::CPR, ITER = BN / ROWS / WAVES;
  static_assert(BN <= 64 && ITER * ROWS * WAVES == BN, "whole instructions");
  uint64_t at[ITER];  // uniform: each instruction's first row, bytes from a head's base
  uint64_t ok;        // the keys that are there: the others are read as zeros

  // One address an instruction, whose rows lie in one cache block (GqaShape::group_rows), made by scalar instructions. (With an address a row for
  // every lane, the addresses alone are 78 vector instructions a tile of 64 keys, a third of the main loop's.)
  __device__ __forceinline__ void place(const GqaArgs& a, const GqaTable& tab, int j0, uint64_t okmask, int wave) {
    ok = okmask;
#pragma unroll
    for (int u = 0; u < ITER; ++u) {
      const int key = j0 + (u * WAVES + wave) * ROWS;
      const uint32_t b = tab.block_at(a, key), t = key - gqa_block_of(a, key) * a.BS;
      at[u] = (uint64_t)b * a.sb_bytes + (uint64_t)t * a.st_bytes;
    }
  }
  // The K (V = false) or V rows straight into LDS. By buffer loads, whose bounds give the zeros; and the
  // compiler takes LDS-direct loads of the global kind for accesses that may return in any order, so that
  // every later LDS read would wait for all reads (lgkmcnt(0)) and some for all loads.
  template <bool V>
  __device__ __forceinline__ void load(const GqaArgs& a, uint8_t* dst, const uint8_t* base, int wave, int lane, int only = -1) const {
    constexpr uint64_t FULL = BN == 64 ? ~0ull : (1ull << (BN & 63)) - 1;
    const int r = lane / G::CPR, c = lane % G::CPR;
    const bool whole = ok == FULL && a.D == G::DL;
#pragma unroll
    for (int u = 0; u < ITER; ++u) {
      if (only >= 0 && u != only) continue;
      const int row = (u * WAVES + wave) * ROWS;
      const int cc = c ^ (V ? G::swz_v(row + r) : G::swz_k(row + r));
      uint32_t off = (uint32_t)r * a.st_bytes + cc * 16;
      if (!whole && !(((uint32_t)(ok >> row) >> r & 1) && cc * G::CE < a.D)) off = 0xFFFFFFFFu;
      const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc((void*)(base + at[u]), (short)0, 0x7FFFFFFF, 0x00020000);
      __builtin_amdgcn_raw_ptr_buffer_load_lds(
          rs, (__attribute__((address_space(3))) void*)(dst + (u * WAVES + wave) * 1024), 16, (int)off, 0, 0, 0);
    }
  }
  // Pools of any alignment and block size, through registers; blk: lane i's is key i's block
  template <bool V>
  __device__ __forceinline__ static void load_any(const GqaArgs& a, uint8_t* dst, const uint8_t* base, int j0, int blk, uint64_t ok,
                                                  int wave, int lane) {
    const int r = lane / G::CPR, c = lane % G::CPR;
#pragma unroll 4
    for (int u = 0; u < ITER; ++u) {
      const int row = (u * WAVES + wave) * ROWS + r, key = j0 + row;
      const int b = __shfl(blk, row, 64);
      const int64_t o = (int64_t)b * a.kv_sb + (int64_t)(key - gqa_block_of(a, key) * a.BS) * a.kv_st;
      const int cc = c ^ (V ? G::swz_v(row) : G::swz_k(row));
      uint4 v = make_uint4(0, 0, 0, 0);
      if ((ok >> row) & 1) v = gqa_chunk<T>(a, reinterpret_cast<const T*>(base) + o, cc * G::CE);
      *reinterpret_cast<uint4*>(dst + (u * WAVES + wave) * 1024 + lane * 16) = v;
    }
  }
};

// A tile's K and V rows into LDS, with the addresses made here.
template <typename T, int DP, int BN, int WAVES, bool VEC>
__device__ __forceinline__ void gqa_fill(const GqaArgs& a, const GqaTable& tab, uint8_t* kt, uint8_t* vt, const uint8_t* kbase,
                                         const uint8_t* vbase, int j0, uint64_t ok, int wave, int lane) {
  using F = GqaFill<T, DP, BN, WAVES>;
  if constexpr (VEC) {
    F f;
    f.place(a, tab, j0, ok, wave);
    if (kt) f.template load<false>(a, kt, kbase, wave, lane);
    if (vt) f.template load<true>(a, vt, vbase, wave, lane);
  } else {
    const int blk = tab.block(a, j0, lane);
    F::template load_any<false>(a, kt, kbase, j0, blk, ok, wave, lane);
    F::template load_any<true>(a, vt, vbase, j0, blk, ok, wave, lane);
  }
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
  // in LDS, since only masked tiles and biased scores need it: the keys [x, y) that a row sees, its
  // position and its slope's bits (times log2(e))
  int4* at;
  int lo_min, lo_max, hi_min, hi_max;  // over the wavefront's rows

  // row0: the wavefront's first packed row of the tile's sequence
  // ranges: 16 NT places of the wavefront's own
  __device__ __forceinline__ void init(const GqaArgs& a, const GqaPlan& p, int row0, int kvh, int4* ranges, int lane) {
    const int g = lane >> 4;
    at = ranges;
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
      int lo, hi, pos;
      gqa_row_range(a, p, tok, lo, hi, pos);
      const float slope = a.slopes ? a.slopes[head] * 1.44269504f : 0.0f;
      if (g == 0) at[16 * n + lane] = make_int4(lo, hi, pos, __float_as_int(slope));
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

  // O^T += V^T P^T over the BN keys in vt (PV), then S = K Q^T for those in kt (QK). The fragments of both
  // are one sequence, read DEPTH ahead of their use: the order is pinned, since the compiler, short of
  // registers, reads each just before its use (a read's latency is four fragments' products; prompt of
  // 8192 so, 2 wavefronts a SIMD taking turns: 972 us).
  template <int BN, bool PV, bool QK, typename F>
  __device__ __forceinline__ void matrix(const uint4 (&pf)[BN / 32 + (BN < 32)][NT], const uint4 (&pr)[BN / 32 + (BN < 32)][NT],
                                         const uint8_t* vt, const uint8_t* kt, f32x4 (&s)[NT][BN / 16], int lane, F beside) {
    constexpr int NV = PV ? BN / 32 * OT : 0, NK = QK ? BN / 16 * QT : 0, N = NV + NK, DEPTH = N < 6 ? N : 6;
    const int g = lane >> 4, c = lane & 15;
    const int vrow = 4 * g + (c >> 2);  // (and 16, 32 further on: the same swizzle)
    const uint8_t* vbase = vt + vrow * G::ROWB + (c & 1) * 8;
    const uint8_t* kbase = kt + c * G::ROWB;
    auto read = [&](int x) __attribute__((always_inline)) {
      if (x < NV) {
        const int h = x / OT, d = x % OT;
        const uint8_t* p = vbase + h * 32 * G::ROWB + (((2 * d + ((c >> 1) & 1)) ^ G::swz_v(vrow)) << 4);
        struct {
          s16x4 a, b;
        } v{__builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)p),
            __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(p + 16 * G::ROWB))};
        return __builtin_bit_cast(uint4, v);
      }
      const int k = (x - NV) % (BN / 16), t = (x - NV) / (BN / 16);  // (a product of the same scores each BN / 16 fragments)
      return *reinterpret_cast<const uint4*>(kbase + k * 16 * G::ROWB + (((4 * t + g) ^ G::swz_k(c)) << 4));
    };
    uint4 f[DEPTH];
#pragma unroll
    for (int x = 0; x < DEPTH; ++x) f[x] = read(x);
#pragma unroll
    for (int x = 0; x < N; ++x) {
      const uint4 v = f[x % DEPTH];
      if (x < NV) {
        const int h = x / OT, d = x % OT;
#pragma unroll
        for (int n = 0; n < NT; ++n) o[n][d] = gqa_mma<T>(v, pf[h][n], o[n][d]);
        if constexpr (SPLIT)
#pragma unroll
          for (int n = 0; n < NT; ++n) o[n][d] = gqa_mma<T>(v, pr[h][n], o[n][d]);
        if (d == OT - 1) {
          constexpr uint32_t ONE = __is_same(T, __bf16) ? 0x3F803F80u : 0x3C003C00u;
          const uint4 ones = make_uint4(ONE, ONE, ONE, ONE);
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            ol[n] = gqa_mma<T>(ones, pf[h][n], ol[n]);
            if constexpr (SPLIT) ol[n] = gqa_mma<T>(ones, pr[h][n], ol[n]);
          }
        }
      } else {
        const int k = (x - NV) % (BN / 16), t = (x - NV) / (BN / 16);
#pragma unroll
        for (int n = 0; n < NT; ++n) s[n][k] = gqa_mma<T>(v, q[n][t], t == 0 ? f32x4{0.f, 0.f, 0.f, 0.f} : s[n][k]);
      }
      if (x + DEPTH < N) f[x % DEPTH] = read(x + DEPTH);
      beside(x);
      __builtin_amdgcn_sched_barrier(0);
    }
  }

  // S = K Q^T for the BN keys in kt
  template <int BN>
  __device__ __forceinline__ void scores(const uint8_t* kt, int lane, f32x4 (&s)[NT][BN / 16]) {
    const uint4 none[BN / 32 + (BN < 32)][NT] = {};
    matrix<BN, false, true>(none, none, nullptr, kt, s, lane, [](int) {});
  }

  // The same from fragments in registers
  template <int KT>
  __device__ __forceinline__ void scores_of(const uint4 (&kf)[KT][QT], f32x4 (&s)[NT][KT]) const {
#pragma unroll
    for (int k = 0; k < KT; ++k) {
#pragma unroll
      for (int n = 0; n < NT; ++n) s[n][k] = gqa_mma<T>(kf[k][0], q[n][0], f32x4{0.f, 0.f, 0.f, 0.f});
#pragma unroll
      for (int t = 1; t < QT; ++t)
#pragma unroll
        for (int n = 0; n < NT; ++n) s[n][k] = gqa_mma<T>(kf[k][t], q[n][t], s[n][k]);
    }
  }

  // Scores -> weights (s becomes P), with the row's state rescaled where its reference moves. okmask: the
  // keys of [j0, j0 + BN) that are there at all. ANYCAP: also caps that need tanh in 16-bit types.
  template <int BN, bool ANYCAP = true>
  __device__ __forceinline__ void weigh(const GqaArgs& a, f32x4 (&s)[NT][BN / 16], int j0, uint64_t okmask, int lane) {
    constexpr int KT = BN / 16;
    // scores in log2 units: s * cc
    float cc = a.c;
    if (!a.simple) {
      cc = 1.0f;
      scored<KT, ANYCAP>(a, s, j0, gqa_here(lane));
    }
    constexpr uint64_t FULL = BN == 64 ? ~0ull : (1ull << (BN & 63)) - 1;
    if (okmask != FULL || !sees_all(j0, BN)) {
      const int here = gqa_here(lane), g = here >> 4;
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        const int4 x = at[16 * n + (here & 15)];
#pragma unroll
        for (int k = 0; k < KT; ++k) {
          const uint32_t there = (uint32_t)(okmask >> (16 * k)) >> (4 * g);
          const int j = j0 + 16 * k + 4 * g;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const bool see = x.x <= j + i && j + i < x.y && ((there >> i) & 1);
            s[n][k][i] = see ? s[n][k][i] : -__builtin_huge_valf();
          }
        }
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
  template <int KT, bool ANYCAP>
  __device__ __forceinline__ void scored(const GqaArgs& a, f32x4 (&s)[NT][KT], int j0, int lane) const {
    if (a.cap > 0.0f && (K::F32 || (ANYCAP && gqa_cap_needs_tanh(a)))) {
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int k = 0; k < KT; ++k)
#pragma unroll
          for (int i = 0; i < 4; ++i) s[n][k][i] = tanhf(s[n][k][i] * a.to_cap) * a.cap;
    } else if (a.cap > 0.0f) {
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int k = 0; k < KT; ++k)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float y = s[n][k][i] * a.to_cap;  // scale / cap
            s[n][k][i] = (1.0f - 2.0f * __builtin_amdgcn_rcpf(__builtin_amdgcn_exp2f(y * 2.88539008f) + 1.0f)) * a.cap;  // cap log2(e)
          }
    } else {
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int k = 0; k < KT; ++k) s[n][k] *= a.c;
    }
    if (a.slopes) {
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        const int4 x = at[16 * n + (lane & 15)];
        const float slope = __int_as_float(x.w);
        const int gap = x.z - j0 - 4 * (lane >> 4);
#pragma unroll
        for (int k = 0; k < KT; ++k)
#pragma unroll
          for (int i = 0; i < 4; ++i) s[n][k][i] = fmaf(-slope, fabsf((float)(gap - (16 * k + i))), s[n][k][i]);
      }
    }
  }

  // O^T += V^T P^T, and the weights' sums
  template <int BN>
  __device__ __forceinline__ void product(f32x4 (&s)[NT][BN / 16], const uint8_t* vt, int lane) {
    if constexpr (K::F32) {
      const int g = lane >> 4, c = lane & 15;
      constexpr int N = BN / 4 * OT, DEPTH = 8;
      auto read = [&](int x) __attribute__((always_inline)) {
        const int i = x / OT % 4, row = 16 * (x / OT / 4) + 4 * g + i, d = x % OT;
        const int ch = (4 * d + (c >> 2)) ^ G::swz_v(row);
        return *reinterpret_cast<const float*>(vt + row * G::ROWB + ch * 16 + (c & 3) * 4);
      };
      float f[DEPTH];
#pragma unroll
      for (int x = 0; x < DEPTH; ++x) f[x] = read(x);
#pragma unroll
      for (int x = 0; x < N; ++x) {
        const float v = f[x % DEPTH];
        const int k = x / OT / 4, i = x / OT % 4, d = x % OT;
#pragma unroll
        for (int n = 0; n < NT; ++n) o[n][d] = __builtin_amdgcn_mfma_f32_16x16x4f32(v, s[n][k][i], o[n][d], 0, 0, 0);
        if (x + DEPTH < N) f[x % DEPTH] = read(x + DEPTH);
        if (x % 4 == 3) __builtin_amdgcn_sched_barrier(0);
      }
    } else {
      uint4 pf[BN / 32][NT], pr[BN / 32][NT];
#pragma unroll
      for (int h = 0; h < BN / 32; ++h)
#pragma unroll
        for (int n = 0; n < NT; ++n) pack(s[n][2 * h], s[n][2 * h + 1], pf[h][n], pr[h][n]);
      matrix<BN, true, false>(pf, pr, vt, nullptr, s, lane, [](int) {});
    }
  }

  // The weights of 32 keys as operands of the product with V
  __device__ __forceinline__ static void pack(const f32x4& x, const f32x4& y, uint4& p, uint4& rest) {
    p = make_uint4(gqa_pack2<T>(x[0], x[1]), gqa_pack2<T>(x[2], x[3]), gqa_pack2<T>(y[0], y[1]), gqa_pack2<T>(y[2], y[3]));
    if constexpr (SPLIT)
      rest = make_uint4(gqa_rest2<T>(x[0], x[1], p.x), gqa_rest2<T>(x[2], x[3], p.y), gqa_rest2<T>(y[0], y[1], p.z),
                        gqa_rest2<T>(y[2], y[3], p.w));
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

// The rows (a bit each) of 16 with a NaN among their sums o, but not in their sum of weights l (a NaN score, which is for all
// elements): V's infinities and NaN times the weight 0 of a row that does not see their key, or of one whose weight is too small for
// its type or has a second part of another sign. (An infinite sum is right: it has no such term.)
template <int OT>
__device__ __forceinline__ uint32_t gqa_odd_rows(const f32x4 (&o)[OT], float l) {
  float z = 0.0f;
#pragma unroll
  for (int d = 0; d < OT; ++d)
#pragma unroll
    for (int i = 0; i < 4; ++i) z += o[d][i];
  uint64_t b = __ballot(z != z && l == l);
  b |= b >> 32;
  return (uint32_t)(b | b >> 16) & 0xFFFFu;
}

// The elements of 16 rows' sums that are NaN in any row: bytes of 1, others 0. By one wavefront, in LDS of its own.
template <int OT>
__device__ __forceinline__ void gqa_odd_elements(const f32x4 (&o)[OT], uint8_t* cols, int lane) {
  for (int e = lane; e < 16 * OT / 4; e += 64) reinterpret_cast<uint32_t*>(cols)[e] = 0;
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
#pragma unroll
  for (int d = 0; d < OT; ++d)
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (o[d][i] != o[d][i]) cols[16 * d + 4 * (lane >> 4) + i] = 1;
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
}

// Bit i: row r0 + i is one of the tile's sequence
__device__ __forceinline__ uint32_t gqa_rows_of(const GqaPlan& p, int r0) {
  return r0 + 16 <= p.rows ? 0xFFFFu : r0 < p.rows ? (1u << (p.rows - r0)) - 1 : 0;
}

// Whether each of the elements marked in `cols` is NaN in a key of [from, to), all of which the 16 rows see. By one wavefront, four
// loads in flight.
template <typename T, int DP>
__device__ __forceinline__ bool gqa_explained(const GqaArgs& a, const GqaPlan& p, const T* vp, const uint8_t* cols, int from, int to, int lane) {
  using G = GqaTile<T, DP>;
  constexpr int ROWS = 64 / G::CPR, CE = G::CE;
  const int c = lane % G::CPR * CE;
  uint32_t left = 0;
#pragma unroll
  for (int e = 0; e < CE; ++e)
    if (c + e < DP && cols[c + e]) left |= 1u << e;
#pragma unroll 1
  for (int j = from; j < to && __any(left != 0); j += 4 * ROWS) {
    uint4 v[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int key = j + u * ROWS + lane / G::CPR, blk = key < to ? p.table[gqa_block_of(a, key)] : -1;
      v[u] = make_uint4(0, 0, 0, 0);
      if (blk >= 0 && blk < a.num_blocks)
        v[u] = gqa_chunk<T>(a, vp + (int64_t)blk * a.kv_sb + (int64_t)(key - gqa_block_of(a, key) * a.BS) * a.kv_st, c);
    }
    left &= ~(gqa_nans<T>(v[0]) | gqa_nans<T>(v[1]) | gqa_nans<T>(v[2]) | gqa_nans<T>(v[3]));
#pragma unroll
    for (int off = G::CPR; off < 64; off <<= 1) left &= __shfl_xor(left, off, 64);
  }
  return !__any(left != 0);
}

// Keys of a step of the second pass below, and the LDS that a wavefront needs for it
template <typename T>
constexpr int gqa_again_wk() { return GqaType<T>::F32 ? 16 : 32; }
template <typename T, int DP>
constexpr int gqa_again_lds() { return gqa_again_wk<T>() * GqaTile<T, DP>::ROWB; }

// The V tile of the keys j .. j + WK in `lds`, as loaded: zeros for infinities and NaN, which are noted in the bits pos and neg (NaN: both) of
// the lane's elements, 4 d + i, where its row sees [lo, hi) of the keys.
template <typename T, int DP>
__device__ __forceinline__ void gqa_clean(uint8_t* lds, int j, int lo, int hi, uint64_t& pos, uint64_t& neg, int lane) {
  using G = GqaTile<T, DP>;
  constexpr int ROWS = 64 / G::CPR, CE = G::CE, ITER = gqa_again_wk<T>() / ROWS;
  const int g = lane >> 4;
#pragma unroll 1
  for (int u = 0; u < ITER; ++u) {
    uint4* at = reinterpret_cast<uint4*>(lds + u * 1024) + lane;
    const uint4 mine = *at;
    const bool odd = gqa_odd_chunk<T>(mine);
    const uint64_t all = __ballot(odd);
    if (all == 0) continue;
#pragma unroll 1
    for (int r = 0; r < ROWS; ++r) {
      if ((all >> (r * G::CPR) & (~0ull >> (64 - G::CPR))) == 0) continue;
      const int row = u * ROWS + r;
      const bool see = lo <= j + row && j + row < hi;
#pragma unroll 1
      for (int d = 0; d < DP / 16; ++d)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int e = 16 * d + 4 * g + i;
          const float f = to_f32(*reinterpret_cast<const T*>(lds + row * G::ROWB + ((e / CE ^ G::swz_v(row)) << 4) + e % CE * (int)sizeof(T)));
          const bool bad = see && !(f * 0.0f == 0.0f);
          pos |= (uint64_t)(bad && !(f < 0.0f)) << (4 * d + i);
          neg |= (uint64_t)(bad && !(f > 0.0f)) << (4 * d + i);
        }
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    if (odd) *at = gqa_finite<T>(mine);
  }
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
}

// The rows of `odd`'s bits, whose sums over the block's keys have NaN elements. Their results are stored already, and right where
// each such element is NaN in a key that all of 16 rows see (`ranges` holds the marks of gqa_odd_elements, 256 bytes for
// each 16 rows). Where not, the 16 rows go over their keys again, with zeros for the infinities and NaN, and these are
// added at the end to the rows that see their keys (a weight is positive: its size does not matter to them). By one
// wavefront, a tile at a time. lds, ranges: the wavefront's own; row_of_tile: its first row's place in the block's tile.
// Arguments and block plan are made anew: those of the kernel, kept from its start to here, cost its loops registers
// and its start their spills (chunks of D = 256 134 -> 160 us, 36 rows of 12 sequences 28 -> 31). For the same reason the calls
// say that they are as good as never reached: the loops in here would count as the kernel's hottest otherwise, and its own
// values be spilled for them (12 sequences of 49 tokens, 4 heads a K/V head, 45.0 us against 41.1).
// Prompt of 2048, 32 heads of 128 over 8, bf16: 111 us; with a NaN in the first token 108, in the last 751 (each such row by
// itself, key by key: 23 ms), NaN alone 117, infinities alone 7.4 ms; prompt of 8192 0.66, 0.72, 6.1 and 120 ms. 64 sequences
// of 2048, a token each: 104 us; a token of NaN 104, one element of it only 500, infinities alone 4.5 ms.
template <typename T, int DP, int NT, bool SPLIT>
__device__ __forceinline__ void gqa_again(uint32_t odd, int row_of_tile, uint8_t* lds, int4* ranges) {
  constexpr int WK = gqa_again_wk<T>();
  const int lane = gqa_here(threadIdx.x & 63);
  int block = blockIdx.x, kvh, split;
  auto* args = (const __attribute__((address_space(4))) GqaArgs*)__builtin_amdgcn_kernarg_segment_ptr();
  asm volatile("" : "+s"(block), "+s"(args));
  const GqaArgs& a = *(const GqaArgs*)args;
  const GqaPlan p = gqa_block_plan(a, block, lane, kvh, split);
  const int row0 = p.row0 + row_of_tile, piece = a.piece0 + split;
  const int from = max(p.lo + (split * p.per << a.bn_log), p.klo), to = min(p.lo + ((split + 1) * p.per << a.bn_log), p.khi);
  using F = GqaFill<T, DP, WK, 1>;
  const T* kp = static_cast<const T*>(a.kp) + kvh * a.kv_sh;
  const T* vp = static_cast<const T*>(a.vp) + kvh * a.kv_sh;
#pragma unroll 1
  for (int n = 0; n < NT; ++n) {
    const uint32_t mine = odd >> (16 * n) & 0xFFFFu;
    if (mine == 0) continue;
    const int r0 = row0 + 16 * n;
    int lo_min, lo_max, hi_min, hi_max;
    gqa_wave_range(a, p, r0, min(r0 + 16, p.rows) - 1, lane, lo_min, lo_max, hi_min, hi_max);
    if (gqa_explained<T, DP>(a, p, vp, reinterpret_cast<const uint8_t*>(ranges + 16 * n), max(from, lo_max), min(to, hi_min), lane)) continue;
    GqaRows<T, DP, 1, SPLIT> rows;
    rows.init(a, p, r0, kvh, ranges, lane);
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    const int4 sees = ranges[lane & 15];  // (the keys [x, y))
    uint64_t pos = 0, neg = 0;
    const int hi = min(to, rows.hi_max);
#pragma unroll 1
    for (int j = max(from, rows.lo_min); j < hi; j += WK) {
      const int blk = lane < WK && j + lane < hi ? p.table[gqa_block_of(a, j + lane)] : -1;
      const uint64_t ok = __ballot(blk >= 0 && blk < a.num_blocks);
      f32x4 s[1][WK / 16];
      F::template load_any<false>(a, lds, reinterpret_cast<const uint8_t*>(kp), j, blk, ok, 0, lane);
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      rows.template scores<WK>(lds, lane, s);
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      F::template load_any<true>(a, lds, reinterpret_cast<const uint8_t*>(vp), j, blk, ok, 0, lane);
      rows.template weigh<WK>(a, s, j, ok, lane);
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      gqa_clean<T, DP>(lds, j, sees.x, sees.y, pos, neg, lane);
      rows.template product<WK>(s, lds, lane);
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    }
    const float l = rows.sum_of(0);
    if (!(mine >> (lane & 15) & 1)) continue;
    const int r = r0 + (lane & 15), tok = p.tok0 + r / a.group, head = kvh * a.group + r % a.group;
#pragma unroll
    for (int d = 0; d < DP / 16; ++d) {
      f32x4 x = rows.o[0][d];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const bool up = pos >> (4 * d + i) & 1, down = neg >> (4 * d + i) & 1;
        if (up || down) x[i] = up && down ? __builtin_nanf("") : up ? __builtin_huge_valf() : -__builtin_huge_valf();
      }
      gqa_store<T>(a, tok, head, piece, p.direct, 16 * d + 4 * (lane >> 4), x, rows.m[0], l);
    }
  }
}

// Many rows: 4 wavefronts of 16 NT rows each share tiles of BN keys, in two LDS buffers.
template <typename T, int DP>
constexpr int gqa_bn() {
  return GqaType<T>::F32 ? (DP <= 64 ? 64 : DP <= 128 ? 32 : 16) : (DP <= 128 ? 64 : 32);
}

template <typename T, int DP, int NT, int BN, bool VEC>
__device__ __forceinline__ void gqa_rows_step(const GqaArgs& a, const GqaTable& tab, GqaRows<T, DP, NT, false>& rows, const uint8_t* __restrict__ cur,
                                              uint8_t* __restrict__ nxt, const uint8_t* __restrict__ kbase,
                                              const uint8_t* __restrict__ vbase, uint64_t ok1, bool now,
                                              bool more, int j0, uint64_t okmask, int wave, int lane) {
  constexpr int TB = BN * GqaTile<T, DP>::ROWB;
  if (more) gqa_fill<T, DP, BN, 4, VEC>(a, tab, nxt, nxt + TB, kbase, vbase, j0 + BN, ok1, wave, lane);
  if (!now || !rows.sees_any(j0, BN)) return;
  f32x4 s[NT][BN / 16];
  rows.template scores<BN>(cur, lane, s);
  rows.template weigh<BN>(a, s, j0, okmask, lane);
  rows.template product<BN>(s, cur + TB, lane);
}

template <typename T, int DP, int NT, bool VEC>
__global__ __launch_bounds__(256, DP <= 128 ? 2 : 1) void gqa_rows_kernel(const GqaArgs a) {
  constexpr int BN = gqa_bn<T, DP>(), TB = BN * GqaTile<T, DP>::ROWB;
  extern __shared__ __align__(1024) uint8_t smem[];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  int kvh, split;
  const GqaPlan p = gqa_block_plan(a, blockIdx.x, lane, kvh, split);
  if (split >= p.live || p.rows <= p.row0) return;
  GqaRows<T, DP, NT, false> rows;
  const int row0 = p.row0 + wave * 16 * NT;
  rows.init(a, p, row0, kvh, reinterpret_cast<int4*>(smem + 4 * TB) + wave * 16 * NT, lane);
  const uint8_t* kbase = static_cast<const uint8_t*>(a.kp) + kvh * a.kv_sh * (int64_t)sizeof(T);
  const uint8_t* vbase = static_cast<const uint8_t*>(a.vp) + kvh * a.kv_sh * (int64_t)sizeof(T);
  const int t0 = split * p.per, t1 = min(p.tiles, t0 + p.per);
  if (t0 < t1) {
    GqaTable tab;
    tab.start(a, p, p.lo + t0 * BN, lane);
    gqa_landed();
    uint64_t ok = 0;
    for (int t = t0 - 1; t < t1; ++t) {  // (the first only loads)
      asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
      uint64_t ok1 = 0;
      if (t + 1 < t1) {
        tab.advance(a, p, p.lo + (t + 1) * BN, lane);
        ok1 = tab.seen<BN>(a, p, p.lo + (t + 1) * BN, lane);
      }
      const int cur = ((t - t0) & 1) * 2 * TB;
      gqa_rows_step<T, DP, NT, BN, VEC>(a, tab, rows, smem + cur, smem + (2 * TB - cur), kbase, vbase, ok1, t >= t0,
                                        t + 1 < t1, p.lo + t * BN, ok, wave, lane);
      ok = ok1;
    }
  }
  const int g = lane >> 4;
  uint32_t odd = 0;  // a bit a row
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    const int r = row0 + 16 * n + (lane & 15);
    const float l = rows.sum_of(n);
    odd |= (gqa_odd_rows(rows.o[n], l) & gqa_rows_of(p, row0 + 16 * n)) << (16 * n);
    if (r < p.rows) {
      const int tok = p.tok0 + r / a.group, head = kvh * a.group + r % a.group;
#pragma unroll
      for (int d = 0; d < DP / 16; ++d)
        gqa_store<T>(a, tok, head, a.piece0 + split, p.direct, 16 * d + 4 * g, rows.o[n][d], rows.m[n], l);
      if (g == 0) gqa_store_live(a, tok, head, split, p.live);
    }
  }
  asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");  // (the tiles are read: their LDS can be used)
  if (__builtin_expect_with_probability(odd == 0, 1, 1.0)) return;
  static_assert(gqa_again_lds<T, DP>() <= TB, "a tile's LDS for each wavefront");
#pragma unroll
  for (int n = 0; n < NT; ++n) gqa_odd_elements(rows.o[n], reinterpret_cast<uint8_t*>(rows.at + 16 * n), lane);
  gqa_again<T, DP, NT, false>(odd, wave * 16 * NT, smem + wave * TB, rows.at);
}

// Many rows of 16-bit types: 8 wavefronts, two a SIMD, in two groups half a step apart: while one
// group's matrix instructions run (the last tile's product with V, this tile's with K), the other
// does its softmax on the vector unit, and a barrier swaps them. Left to themselves the two
// wavefronts of a SIMD overlap by chance only (prompt of 8192, 32 heads of 128 over 8, 4 wavefronts a block:
// 649 us, matrix unit busy 36%, vector unit 41%).
// K and V tiles go through rings of 3: tile i + 2 of K and i + 1 of V are loaded from the start of step i.
template <typename T, int DP>
constexpr int gqa_pair_bn() { return DP <= 128 ? 64 : 32; }

template <typename T, int DP, int NT>
struct GqaPair {
  static constexpr int BN = gqa_pair_bn<T, DP>(), TB = BN * GqaTile<T, DP>::ROWB, PER = TB / 1024 / 8;
  static constexpr int RANGES = 6 * TB > 8 * gqa_again_lds<T, DP>() ? 6 * TB : 8 * gqa_again_lds<T, DP>();  // rows' ranges, behind the tiles
  using Fill = GqaFill<T, DP, BN, 8>;
  GqaRows<T, DP, NT, false> rows;
  f32x4 s[NT][BN / 16];
  uint4 pf[BN / 32][NT];

  // kr, vr: tiles i of K, i - 1 of V; kw, vw: the slots of tiles i + 2 and i + 1. (Every pointer is __restrict, the loads' sources
  // too, or the loads would hold up the reads; no wait is in here, since one would not order accesses through them.)
  __device__ __forceinline__ void multiply(const GqaArgs& a, const uint8_t* __restrict__ kr, uint8_t* __restrict__ kw,
                                           const uint8_t* __restrict__ vr, uint8_t* __restrict__ vw,
                                           const uint8_t* __restrict__ kbase, const uint8_t* __restrict__ vbase,
                                           const Fill& kat, const Fill& vat, bool kmore, bool vmore, int wave, int lane) {
    // The loads go between the fragments (at the head of the step: prompt of 8192, 565 us against 550), but in the
    // widest heads, whose tiles' products are as many for half the keys (chunks of D = 256: 139 against 152).
    constexpr bool BETWEEN = DP <= 128;
    if (!BETWEEN && vmore) vat.template load<true>(a, vw, vbase, wave, lane);
    if (!BETWEEN && kmore) kat.template load<false>(a, kw, kbase, wave, lane);
    rows.template matrix<BN, true, true>(pf, pf, vr, kr, s, lane, [&](int x) __attribute__((always_inline)) {
#pragma unroll
      for (int u = 0; u < PER && BETWEEN; ++u) {
        if (x == 4 + 8 * u && vmore) vat.template load<true>(a, vw, vbase, wave, lane, u);
        if (x == 8 + 8 * u && kmore) kat.template load<false>(a, kw, kbase, wave, lane, u);
      }
    });
  }
  __device__ __forceinline__ void soften(const GqaArgs& a, int j0, uint64_t okmask, int lane) {
    rows.template weigh<BN, false>(a, s, j0, okmask, lane);
    uint4 none;
#pragma unroll
    for (int h = 0; h < BN / 32; ++h)
#pragma unroll
      for (int n = 0; n < NT; ++n) GqaRows<T, DP, NT, false>::pack(s[n][2 * h], s[n][2 * h + 1], pf[h][n], none);
  }
};

template <typename T, int DP, int NT>
__global__ __launch_bounds__(512, 2) void gqa_pair_kernel(const GqaArgs a) {
  using P = GqaPair<T, DP, NT>;
  constexpr int BN = P::BN, TB = P::TB;
  extern __shared__ __align__(1024) uint8_t smem[];  // 3 tiles of K, 3 of V
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  int kvh, split;
  const GqaPlan p = gqa_block_plan(a, blockIdx.x, lane, kvh, split);
  if (split >= p.live || p.rows <= p.row0) return;
  const uint8_t* kbase = static_cast<const uint8_t*>(a.kp) + kvh * a.kv_sh * (int64_t)sizeof(T);
  const uint8_t* vbase = static_cast<const uint8_t*>(a.vp) + kvh * a.kv_sh * (int64_t)sizeof(T);
  const int t0 = split * p.per, n = min(p.tiles - t0, p.per), j0 = p.lo + t0 * BN;
  P w;
  const int row0 = p.row0 + wave * 16 * NT;
  w.rows.init(a, p, row0, kvh, reinterpret_cast<int4*>(smem + P::RANGES) + wave * 16 * NT, lane);
  if (n > 0) {
    GqaTable tab;
    tab.start(a, p, j0, lane);
    gqa_landed();
    typename P::Fill f1, f2;  // tiles i + 1 and i + 2
    uint64_t ok0 = tab.seen<BN>(a, p, j0, lane);
    gqa_fill<T, DP, BN, 8, true>(a, tab, smem, smem + 3 * TB, kbase, vbase, j0, ok0, wave, lane);
    auto place = [&](typename P::Fill& f, int i) __attribute__((always_inline)) {
      if (i < n) {
        tab.advance(a, p, j0 + i * BN, lane);
        f.place(a, tab, j0 + i * BN, tab.seen<BN>(a, p, j0 + i * BN, lane), wave);
      }
    };
    place(f1, 1);
    if (n > 1) f1.template load<false>(a, smem + TB, kbase, wave, lane);
    place(f2, 2);
    // V's tile -1: zeros, with weights of 0
    for (int e = threadIdx.x; e < TB / 16; e += 512) reinterpret_cast<uint4*>(smem + 5 * TB)[e] = make_uint4(0, 0, 0, 0);
#pragma unroll
    for (int h = 0; h < BN / 32; ++h)
#pragma unroll
      for (int m = 0; m < NT; ++m) w.pf[h][m] = make_uint4(0, 0, 0, 0);
    gqa_landed();
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
    if (wave >= 4) asm volatile("s_barrier" ::: "memory");  // half a step behind
    int s0 = 0, s1 = TB, s2 = 2 * TB;  // slots of tiles i, i + 1, i + 2 (and so of i - 1)
    for (int i = 0; i < n; ++i) {
      __builtin_amdgcn_s_setprio(1);  // (its matrix instructions before the other's exponentials: 620 us without)
      w.multiply(a, smem + s0, smem + s2, smem + 3 * TB + s2, smem + 3 * TB + s1, kbase, vbase, f2, f1, i + 2 < n,
                 i + 1 < n, wave, lane);
      __builtin_amdgcn_s_setprio(0);
      // the last step's loads have landed (this one's may be on their way)
      if (i + 2 < n) asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(2 * P::PER) : "memory");
      else asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
      w.soften(a, j0 + i * BN, ok0, lane);
      const int t = s0;
      s0 = s1, s1 = s2, s2 = t;
      ok0 = f1.ok;
      f1 = f2;
      place(f2, i + 3);  // (here and not among the products, which are what a step waits for)
      asm volatile("s_barrier" ::: "memory");
    }
    w.rows.template matrix<BN, true, false>(w.pf, w.pf, smem + 3 * TB + s2, nullptr, w.s, lane, [](int) {});
    if (!(wave >= 4)) asm volatile("s_barrier" ::: "memory");
  }
  const int g = lane >> 4;
  uint32_t odd = 0;  // a bit a row
#pragma unroll
  for (int m = 0; m < NT; ++m) {
    const int r = row0 + 16 * m + (lane & 15);
    const float l = w.rows.sum_of(m);
    odd |= (gqa_odd_rows(w.rows.o[m], l) & gqa_rows_of(p, row0 + 16 * m)) << (16 * m);
    if (r < p.rows) {
      const int tok = p.tok0 + r / a.group, head = kvh * a.group + r % a.group;
#pragma unroll
      for (int d = 0; d < DP / 16; ++d)
        gqa_store<T>(a, tok, head, a.piece0 + split, p.direct, 16 * d + 4 * g, w.rows.o[m][d], w.rows.m[m], l);
      if (g == 0) gqa_store_live(a, tok, head, split, p.live);
    }
  }
  asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");  // (the tiles are read: their LDS can be used)
  if (__builtin_expect_with_probability(odd == 0, 1, 1.0)) return;
#pragma unroll
  for (int m = 0; m < NT; ++m) gqa_odd_elements(w.rows.o[m], reinterpret_cast<uint8_t*>(w.rows.at + 16 * m), lane);
  gqa_again<T, DP, NT, false>(odd, wave * 16 * NT, smem + wave * gqa_again_lds<T, DP>(), w.rows.at);
}

// Few rows: the NW wavefronts of a block hold the same 16 rows and take WK keys each of a
// step of NW WK keys, so that no wavefront waits for another before the end, where their states are
// joined through LDS. K's fragments are loaded straight into registers (16 rows of 64 bytes an
// instruction), the next tile's as soon as this one's scores are made; V tiles go through LDS, to be read
// transposed, the next one's loads issued after this one's product. (With two K and two V buffers in LDS and
// 4 wavefronts a CU: 40 sequences of 1 to 4096 tokens, 32 heads of 128 over 8 K/V heads, 45 us; so 35. 64 of 2048: 104,
// 5.2 TB/s.) What a block takes before its first key (lengths, table, keys: three loads one after the other, 7 us by its clock) is
// most of what short contexts take, and code that runs once costs as much as the loads: it is fetched anew in each launch.
template <typename T, int DP>
constexpr int gqa_wk() { return GqaType<T>::F32 ? (DP <= 64 ? 32 : 16) : 32; }
template <typename T, int DP>
constexpr int gqa_nw() { return gqa_wk<T, DP>() * GqaTile<T, DP>::ROWB > 8192 ? 2 : 4; }

// The K fragments of keys j0 .. j0 + 16 KT; blk: lane i's is key i's block.
template <typename T, int DP, int KT>
__device__ __forceinline__ void gqa_load_k(const GqaArgs& a, uint4 (&kf)[KT][DP / (4 * GqaType<T>::CE)], const uint8_t* base, int j0,
                                           int blk, uint64_t ok, int lane) {
  constexpr int CE = GqaType<T>::CE, QT = DP / (4 * CE);
  const int g = lane >> 4, c = lane & 15;
  const uint8_t* zero = reinterpret_cast<const uint8_t*>(gqa_zeros) + g * 16;
#pragma unroll
  for (int k = 0; k < KT; ++k) {
    const int b = __shfl(blk, 16 * k + c, 64), key = j0 + 16 * k + c;
    const int64_t o = ((int64_t)b * a.kv_sb + (int64_t)(key - gqa_block_of(a, key) * a.BS) * a.kv_st) * (int64_t)sizeof(T);
    const uint8_t* row = (ok >> (16 * k + c)) & 1 ? base + o + g * 16 : zero;
#pragma unroll
    for (int t = 0; t < QT; ++t) {
      const uint8_t* from = a.D == DP || (4 * t + g) * CE < a.D ? row : zero;
      // (said to be global memory: chosen between two pointers, it would be a load of the flat kind)
      kf[k][t] = __builtin_bit_cast(
          uint4, __builtin_nontemporal_load((const __attribute__((address_space(1))) i32x4*)(from + t * 64)));
    }
  }
}

template <typename T, int DP>
__global__ __launch_bounds__((gqa_nw<T, DP>() * 64), (gqa_nw<T, DP>() / 2)) void gqa_keys_kernel(const GqaArgs a) {
  constexpr int NT = 1;
  constexpr int WK = gqa_wk<T, DP>(), NW = gqa_nw<T, DP>(), TB = WK * GqaTile<T, DP>::ROWB, BN = NW * WK;
  constexpr int OL = DP + 4;  // floats of an output row in LDS
  extern __shared__ __align__(1024) uint8_t smem[];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  int kvh, split;
  const GqaPlan p = gqa_block_plan(a, blockIdx.x, lane, kvh, split);
  if (split >= p.live || p.rows <= p.row0) return;
  GqaRows<T, DP, NT, !GqaType<T>::F32> rows;
  const uint8_t* kbase = static_cast<const uint8_t*>(a.kp) + kvh * a.kv_sh * (int64_t)sizeof(T);
  const uint8_t* vbase = static_cast<const uint8_t*>(a.vp) + kvh * a.kv_sh * (int64_t)sizeof(T);
  int t0 = split * p.per, t1 = min(p.tiles, t0 + p.per);
  // this wavefront's first and last steps may hold none of its keys
  if (p.lo + t0 * BN + (wave + 1) * WK <= p.klo) ++t0;
  t1 = min(t1, (p.khi - p.lo - wave * WK + BN - 1) / BN);
  uint8_t* vt = smem + wave * TB;
  auto first = [&](int t) { return p.lo + t * BN + wave * WK; };
  GqaTable tab;
  rows.init(a, p, p.row0, kvh, reinterpret_cast<int4*>(smem + NW * TB) + wave * 16 * NT, lane);
  if (t0 < t1) tab.start(a, p, first(t0), lane);
  gqa_landed();
  uint64_t ok = 0;
  if (t0 < t1) {
    constexpr int KT = WK / 16, PER = KT * (DP / (4 * GqaType<T>::CE));  // loads of a K tile
    uint4 kf[KT][DP / (4 * GqaType<T>::CE)];
    ok = tab.seen<WK>(a, p, first(t0), lane);
    gqa_load_k<T, DP, KT>(a, kf, kbase, first(t0), tab.block(a, first(t0), lane), ok, lane);
    gqa_fill<T, DP, WK, 1, true>(a, tab, nullptr, vt, nullptr, vbase, first(t0), ok, 0, lane);
    for (int t = t0; t < t1 - 1; ++t) {
      tab.advance(a, p, first(t + 1), lane);
      const uint64_t ok1 = tab.seen<WK>(a, p, first(t + 1), lane);
      f32x4 s[NT][KT];
      rows.scores_of(kf, s);
      gqa_load_k<T, DP, KT>(a, kf, kbase, first(t + 1), tab.block(a, first(t + 1), lane), ok1, lane);
      rows.template weigh<WK>(a, s, first(t), ok, lane);
      // loads complete in order: this V tile's are older than the K fragments'
      asm volatile("s_waitcnt vmcnt(%0)" ::"n"(PER) : "memory");
      rows.template product<WK>(s, vt, lane);
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // (V is read)
      gqa_fill<T, DP, WK, 1, true>(a, tab, nullptr, vt, nullptr, vbase, first(t + 1), ok1, 0, lane);
      ok = ok1;
    }
    f32x4 s[NT][KT];
    rows.scores_of(kf, s);
    rows.template weigh<WK>(a, s, first(t1 - 1), ok, lane);
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    rows.template product<WK>(s, vt, lane);
  }
  // join the wavefronts' states
  float* ol = reinterpret_cast<float*>(smem);                // [NW][16 NT][OL]
  float* ml = ol + NW * 16 * NT * OL;                        // [NW][16 NT][2]
  uint32_t* odd = reinterpret_cast<uint32_t*>(ml + NW * 16 * NT * 2);  // [NW]: rows with NaN sums
  __syncthreads();
  uint32_t mine = 0;
  const int g = lane >> 4;
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    const int r = 16 * n + (lane & 15);
    const float l = rows.sum_of(n);
    mine |= (gqa_odd_rows(rows.o[n], l) & gqa_rows_of(p, p.row0 + 16 * n)) << (16 * n);
#pragma unroll
    for (int d = 0; d < DP / 16; ++d)
      *reinterpret_cast<f32x4*>(ol + (wave * 16 * NT + r) * OL + 16 * d + 4 * g) = rows.o[n][d];
    if (g == 0) *reinterpret_cast<float2*>(ml + (wave * 16 * NT + r) * 2) = make_float2(rows.m[n], l);
  }
  if (lane == 0) odd[wave] = mine;
  __syncthreads();
  uint32_t all = 0;
#pragma unroll
  for (int w = 0; w < NW; ++w) all |= __builtin_amdgcn_readfirstlane(odd[w]);
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
  if (__builtin_expect_with_probability(all == 0, 1, 1.0)) return;
  asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");  // (results are stored, their LDS is read)
  static_assert(gqa_again_lds<T, DP>() <= TB, "a tile's LDS");
  if (wave != 0) return;
  // (which elements are NaN is not kept: all count, as a token that is no number makes them)
  for (int e = lane; e < DP; e += 64) reinterpret_cast<uint8_t*>(rows.at)[e] = e < a.D;
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  gqa_again<T, DP, NT, !GqaType<T>::F32>(all, 0, smem, rows.at);
}

template <typename T, int DP>
constexpr int gqa_keys_lds() {
  constexpr int NW = gqa_nw<T, DP>();
  constexpr int tiles = NW * (gqa_wk<T, DP>() * GqaTile<T, DP>::ROWB + 256), join = NW * 16 * (DP + 4 + 2) * 4 + 4 * NW;
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
  if (s.keys) return gqa_launch_kernel<gqa_keys_kernel<T, DP>>(a, blocks, gqa_nw<T, DP>() * 64, gqa_keys_lds<T, DP>(), st);
  if constexpr (!GqaType<T>::F32) {
    if (s.pair) {
      constexpr int NT = DP <= 128 ? 2 : 1;
      return gqa_launch_kernel<gqa_pair_kernel<T, DP, NT>>(a, blocks, 512, GqaPair<T, DP, NT>::RANGES + 8 * 256 * NT, st);
    }
  }
  constexpr int lds = 4 * gqa_bn<T, DP>() * GqaTile<T, DP>::ROWB + 4 * 256 * 2;
  if (!s.vec) return gqa_launch_kernel<gqa_rows_kernel<T, DP, 1, false>>(a, blocks, 256, lds, st);
  if constexpr (GqaType<T>::F32)
    if (s.nt == 2) return gqa_launch_kernel<gqa_rows_kernel<T, DP, 2, true>>(a, blocks, 256, lds, st);
  return gqa_launch_kernel<gqa_rows_kernel<T, DP, 1, true>>(a, blocks, 256, lds, st);
}

template <typename T, int DP>
void gqa_tiles_dp(GqaShape& s) {
  s.bn = s.keys ? gqa_nw<T, DP>() * gqa_wk<T, DP>() : s.pair ? gqa_pair_bn<T, DP>() : gqa_bn<T, DP>();
  s.group_rows = 64 / GqaTile<T, DP>::CPR;
  s.bm = s.keys ? 16 : s.pair ? (DP <= 128 ? 256 : 128) : 64 * s.nt;
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
