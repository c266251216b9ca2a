// Tiles of a product of two matrices whose rows both run along the reduction axis: the int8 products (gemm_a8.hip) and, turned
// first, the weight gradients (gemm_dw8.hip). Two ways to run one: large tiles by two groups of wavefronts half a step apart (NtTile), small ones
// by wavefronts that multiply beside others that load (NtSmall); and the choice between their sizes (nt_choose).
//
// Op: the matrix instruction of 16 rows by 16 rows over 64 bytes of each (int8: 64 values, 16-bit types: 32):
// Acc and mma(first, second, acc). Lane (lr, lk) = (lane & 15, lane >> 4) gives row lr's 16-byte chunk lk of both and
// ends with the products of second's row lr and first's rows 4 lk .. 4 lk + 3.
//
// NtTile. A block is 8 wavefronts on a tile of B x B, group g = wavefronts 4 g .. 4 g + 3, one of each group on every SIMD. A step is 64 bytes
// of every row. In phase 2 s + g group g moves step s from LDS to registers, in the next phase it multiplies, and the other group
// does the opposite: the matrix cores always have a wavefront whose operands are there. A barrier ends a phase.
//
// A stage is two steps: 128 bytes of every row, whole cache lines (64 bytes a row and load: twice the requests, and L2 gives half as
// much). LDS holds NB stages, filled by loads that write it directly, group 0 a's rows, group 1 b's. Stage t + NB - 1 is asked for
// from phase 4 t on, when the last read of stage t - 1 is over, and waited for at the end of phase 4 (t + NB - 1) - 1, the last
// before it is read. (Measured, int8 4096 x 8192 x 8192, single launches traced: 198 to
// 212 us by box, 2.6 to 2.8 POP/s, matrix cores busy 67%; call upon call, at the clock that is left then, 226 to 231; all wavefronts in step with
// two buffers 277 where this took 248.)
//
// Row r's chunk c of a stage lies in slot r * 8 + (c ^ (r & 7)): the 16 rows of an operand cover all banks. Loads write
// lane l's chunk to slot base + l, so each lane loads the chunk that belongs there.
#pragma once

#include "common.h"

namespace mls {

constexpr int kNtOutside = (int)0x80000000u;  // past every descriptor (they span < 2^31 bytes)

struct NtOperands {
  const uint8_t* a;  // [M][lda] bytes
  const uint8_t* b;  // [N][ldb]
  int lda, ldb;      // bytes, multiples of 16, as a and b
  int M, N, K;       // K: bytes of a row, a multiple of 16
  int turns = 1;     // a's rows are that many parts of K / turns bytes, a multiple of 128 where there are several; each meets the same row of b
};

// The rows first .. first + rows of a matrix. The offsets that lanes give are checked against it.
__device__ __forceinline__ __amdgpu_buffer_rsrc_t nt_rows(const void* base, int64_t first, int64_t ld, int rows, int K) {
  return __builtin_amdgcn_make_buffer_rsrc((void*)((const uint8_t*)base + first * ld), (short)0, (int)((rows - 1) * ld + K),
                                           0x00020000);
}

__device__ __forceinline__ void nt_lds_load16(__amdgpu_buffer_rsrc_t rs, void* lds, int voff) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (__attribute__((address_space(3))) void*)lds, 16, voff, 0, 0, 0);
}

// The stage of b that stage t of a meets; part: stages a part, or a large number.
__device__ __forceinline__ int nt_stage_of_b(int t, int part) { return t < part ? t : t < 2 * part ? t - part : t - 2 * part; }
__device__ __forceinline__ int nt_part(const NtOperands& p) { return p.turns == 1 ? 0x3FFFFFFF : p.K / p.turns / 128; }

// Block -> (K range, row tile, column tile): consecutive tiles on one XCD, runs of 4 row tiles sweep all
// column tiles.
__device__ __forceinline__ void nt_place(int m_tiles, int n_tiles, int& split, int& mt, int& nt) {
  constexpr int GM = 4;
  const int L = xcd_remap(blockIdx.x, gridDim.x), tiles = m_tiles * n_tiles;
  split = L / tiles;
  const int t = L - split * tiles, per = GM * n_tiles, first = t / per * GM, size = min(m_tiles - first, GM), r = t % per;
  mt = first + r % size;
  nt = r / size;
}

// One step's operands of a wavefront from LDS, waited for: a's 16-row tiles lie 2048 bytes apart from address
// `a`, b's from `b`. (One statement with its wait: the compiler would hold plain reads behind every load to LDS in flight.)
template <int TM, int TN>
__device__ __forceinline__ void nt_read(uint32_t a, uint32_t b, i32x4 (&x)[TM], i32x4 (&y)[TN]) {
  static_assert((TM == 8 && TN == 4) || (TM == 4 && TN == 2), "a half by a quarter of a square");
  if constexpr (TM == 8) {
    asm volatile(
        "ds_read_b128 %8, %13\n\tds_read_b128 %0, %12\n\tds_read_b128 %9, %13 offset:2048\n\t"
        "ds_read_b128 %10, %13 offset:4096\n\tds_read_b128 %11, %13 offset:6144\n\t"
        "ds_read_b128 %1, %12 offset:2048\n\tds_read_b128 %2, %12 offset:4096\n\tds_read_b128 %3, %12 offset:6144\n\t"
        "ds_read_b128 %4, %12 offset:8192\n\tds_read_b128 %5, %12 offset:10240\n\tds_read_b128 %6, %12 offset:12288\n\t"
        "ds_read_b128 %7, %12 offset:14336\n\ts_waitcnt lgkmcnt(0)"
        : "=&v"(x[0]), "=&v"(x[1]), "=&v"(x[2]), "=&v"(x[3]), "=&v"(x[4]), "=&v"(x[5]), "=&v"(x[6]), "=&v"(x[7]), "=&v"(y[0]),
          "=&v"(y[1]), "=&v"(y[2]), "=&v"(y[3])
        : "v"(a), "v"(b)
        : "memory");
  } else {
    asm volatile(
        "ds_read_b128 %4, %7\n\tds_read_b128 %0, %6\n\tds_read_b128 %5, %7 offset:2048\n\tds_read_b128 %1, %6 offset:2048\n\t"
        "ds_read_b128 %2, %6 offset:4096\n\tds_read_b128 %3, %6 offset:6144\n\ts_waitcnt lgkmcnt(0)"
        : "=&v"(x[0]), "=&v"(x[1]), "=&v"(x[2]), "=&v"(x[3]), "=&v"(y[0]), "=&v"(y[1])
        : "v"(a), "v"(b)
        : "memory");
  }
}

template <class Op, int B, int NB>
struct NtTile {
  static constexpr int BM = B, BN = B, THREADS = 512;
  static constexpr bool RANGES = false;  // (whether it is run on ranges of K)
  static constexpr int WTM = B / 2, WTN = B / 4, TM = WTM / 16, TN = WTN / 16;
  static constexpr int STAGE = 2 * B * 128;  // bytes
  static constexpr int LDS = NB * STAGE;
  static constexpr int PW = B * 8 / 256;     // loads of 64 chunks a wavefront and stage
  static_assert(B % 64 == 0 && NB >= 2 && (NB - 2) * PW < 64, "whole loads, and a count that vmcnt holds");
  using Acc = typename Op::Acc;

  __device__ static __forceinline__ void phase_end() {
    __builtin_amdgcn_sched_barrier(0);
    asm volatile("s_barrier" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
  }

  // Stages k_lo .. k_hi of 128 bytes of the tile at (m0, n0), in `lds` of LDS bytes. acc[i][j]: b's rows
  // 16 i .. of this wavefront's WTN, a's 16 j .. of its WTM.
  __device__ static __forceinline__ bool run(const NtOperands& p, uint8_t* lds, int m0, int n0, int k_lo, int k_hi, int wave, int lane,
                                             Acc (&acc)[TN][TM]) {
    const int g = wave >> 2, w = wave & 3;
    const __amdgpu_buffer_rsrc_t rs = g == 0 ? nt_rows(p.a, m0, p.lda, min(B, p.M - m0), p.K) : nt_rows(p.b, n0, p.ldb, min(B, p.N - n0), p.K / p.turns);
    const int ld = g == 0 ? p.lda : p.ldb;
    const int lc = ((lane & 7) ^ ((lane >> 3) & 7)) * 16;  // (a load's 8 rows begin at a multiple of 8)
    const int off = (w * PW * 8 + (lane >> 3)) * ld + lc;
    uint8_t* const fill = lds + (g * B + w * PW * 8) * 128;
    const int part = g == 0 ? 0x3FFFFFFF : nt_part(p);
    // where this lane's first chunk of stage t lies; past K, and past the last stage: outside, and the loads write zeros and
    // read no memory (so are the chunks of the rows below it: 256 rows span less than 2^31 bytes)
    auto start = [&](int t) __attribute__((always_inline)) {
      return t < k_hi && t * 128 + lc < p.K ? off + nt_stage_of_b(t, part) * 128 : kNtOutside;
    };
    auto ask = [&](int i, int at, int buf) __attribute__((always_inline)) {
      nt_lds_load16(rs, fill + buf * STAGE + i * 1024, at + i * 8 * ld);
    };
#pragma unroll
    for (int i = 0; i < TN; ++i)
#pragma unroll
      for (int j = 0; j < TM; ++j) acc[i][j] = Acc{0, 0, 0, 0};

    const int lr = lane & 15, lk = lane >> 4;
    const uint32_t base = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint8_t*)lds + lr * 128 + (lk ^ (lr & 7)) * 16;
    const uint32_t at_a = base + g * WTM * 128, at_b = base + (B + w * WTN) * 128;

    constexpr int left = (NB - 2) * PW;  // loads of later stages
    constexpr int wait_code = (left & 15) | (left >> 4) << 14 | 0x70 | 0xF00;
    for (int t = 0; t < NB - 1; ++t)
#pragma unroll
      for (int i = 0; i < PW; ++i) ask(i, start(k_lo + t), t);
    __builtin_amdgcn_s_waitcnt(wait_code);
    phase_end();
    if (g == 1) phase_end();  // half a step later
    int buf = 0;
    for (int t = k_lo; t < k_hi; ++t) {
      const int last = buf == 0 ? NB - 1 : buf - 1, at = start(t + NB - 1);
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        i32x4 x[TM], y[TN];
        nt_read<TM, TN>((at_a + buf * STAGE) ^ (h * 64), (at_b + buf * STAGE) ^ (h * 64), x, y);
        if (h == 1 && g == 1) __builtin_amdgcn_s_waitcnt(wait_code);
        // half of the next stage's loads behind the first step's reads, half among its products: all of them at one place
        // hold up that phase
        if (h == 0) {
          __builtin_amdgcn_sched_barrier(0);
#pragma unroll
          for (int i = 0; i < PW / 2; ++i) ask(i, at, last);
        }
        phase_end();
        __builtin_amdgcn_s_setprio(1);
#pragma unroll
        for (int j = 0; j < TM; ++j) {
#pragma unroll
          for (int i = 0; i < TN; ++i) acc[i][j] = Op::mma(y[i], x[j], acc[i][j]);
          if (h == 0 && j < PW - PW / 2) {
            __builtin_amdgcn_sched_barrier(0);
            ask(PW / 2 + j, at, last);
            __builtin_amdgcn_sched_barrier(0);
          }
        }
        __builtin_amdgcn_s_setprio(0);
        __builtin_amdgcn_sched_barrier(0);
        if (h == 1 && g == 0) __builtin_amdgcn_s_waitcnt(wait_code);
        phase_end();
      }
      buf = buf == NB - 1 ? 0 : buf + 1;
    }
    if (g == 0) phase_end();
    __builtin_amdgcn_s_waitcnt(0x70 | 0xF00);  // no load writes LDS after the block
    return true;
  }

  // This wavefront's first output: the lane holds, in acc[i][j][e], row + 16 j and column + 16 i + e.
  __device__ static __forceinline__ int row(int m0, int wave, int lane) { return m0 + (wave >> 2) * WTM + (lane & 15); }
  __device__ static __forceinline__ int column(int n0, int wave, int lane) { return n0 + (wave & 3) * WTN + 4 * (lane >> 4); }
};

// Outputs of two neighbouring tiles of 16 columns, 16-bit: lane (lr, lk) holds columns 4 lk .. 4 lk + 3 of both (lo: those
// of the first). Odd and even lk trade halves (v_permlane16_swap), so that a lane stores 16 bytes, and a row's 4 lanes 64 in
// one instruction. `row`: of the first column of the first tile, n: that column; wide: rows are 16-byte aligned.
__device__ __forceinline__ void nt_store_pair(uint16_t* row, int n, int N, uint2 lo, uint2 hi, int lk, bool in, bool wide) {
  const auto x = __builtin_amdgcn_permlane16_swap(lo.x, hi.x, false, false);
  const uint32_t x0 = x[0], x1 = x[1];
  const auto y = __builtin_amdgcn_permlane16_swap(lo.y, hi.y, false, false);
  const uint32_t y0 = y[0], y1 = y[1];
  const int c = 16 * (lk & 1) + 8 * (lk >> 1);
  if (!in || n + c >= N) return;
  if (wide && n + c + 8 <= N) {
    *reinterpret_cast<uint4*>(row + c) = make_uint4(x0, y0, x1, y1);
  } else {
    const uint32_t w[4] = {x0, y0, x1, y1};
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (n + c + e < N) row[c + e] = (uint16_t)(w[e / 2] >> (16 * (e % 2)));
  }
}

// Both steps' operands of a stage, waited for: a's 16-row tiles lie 2048 bytes apart from address `a`, b's from `b`.
template <int TM, int TN>
__device__ __forceinline__ void nt_read_stage(uint32_t a, uint32_t b, i32x4 (&x)[2][TM], i32x4 (&y)[2][TN]) {
  static_assert((TM == 4 && TN == 2) || (TM == 2 && TN == 2), "32 or 64 rows by 32");
  if constexpr (TM == 4) {
    asm volatile(
        "ds_read_b128 %8, %14\n\tds_read_b128 %9, %14 offset:2048\n\t"
        "ds_read_b128 %0, %12\n\tds_read_b128 %1, %12 offset:2048\n\t"
        "ds_read_b128 %2, %12 offset:4096\n\tds_read_b128 %3, %12 offset:6144\n\t"
        "ds_read_b128 %10, %15\n\tds_read_b128 %11, %15 offset:2048\n\t"
        "ds_read_b128 %4, %13\n\tds_read_b128 %5, %13 offset:2048\n\t"
        "ds_read_b128 %6, %13 offset:4096\n\tds_read_b128 %7, %13 offset:6144\n\t"
        "s_waitcnt lgkmcnt(0)"
        : "=&v"(x[0][0]), "=&v"(x[0][1]), "=&v"(x[0][2]), "=&v"(x[0][3]), "=&v"(x[1][0]), "=&v"(x[1][1]), "=&v"(x[1][2]),
          "=&v"(x[1][3]), "=&v"(y[0][0]), "=&v"(y[0][1]), "=&v"(y[1][0]), "=&v"(y[1][1])
        : "v"(a), "v"(a ^ 64), "v"(b), "v"(b ^ 64)
        : "memory");
  } else {
    asm volatile(
        "ds_read_b128 %4, %10\n\tds_read_b128 %5, %10 offset:2048\n\t"
        "ds_read_b128 %0, %8\n\tds_read_b128 %1, %8 offset:2048\n\t"
        "ds_read_b128 %6, %11\n\tds_read_b128 %7, %11 offset:2048\n\t"
        "ds_read_b128 %2, %9\n\tds_read_b128 %3, %9 offset:2048\n\t"
        "s_waitcnt lgkmcnt(0)"
        : "=&v"(x[0][0]), "=&v"(x[0][1]), "=&v"(x[1][0]), "=&v"(x[1][1]), "=&v"(y[0][0]), "=&v"(y[0][1]), "=&v"(y[1][0]),
          "=&v"(y[1][1])
        : "v"(a), "v"(a ^ 64), "v"(b), "v"(b ^ 64)
        : "memory");
  }
}

// NtSmall. The same product on a tile of BM x BN, one barrier a stage: CW wavefronts of 2 x CW / 2 multiply, LW more only load. A
// wavefront's load of 64 chunks takes about 40 ns to go out, whatever comes of it, so that loads in front of a
// small tile's few products would take longer than they (64 x 64: 255 ns a stage; with loaders 140 to 180).
template <class Op, int BM_, int BN_, int NB, int CW, int LW>
struct NtSmall {
  static constexpr int BM = BM_, BN = BN_, THREADS = 64 * (CW + LW);
  static constexpr bool RANGES = true;
  static constexpr int WN = CW / 2, WTM = BM / 2, WTN = BN / WN, TM = WTM / 16, TN = WTN / 16;
  static constexpr int STAGE = (BM + BN) * 128, LDS = NB * STAGE;
  static constexpr int PW = (BM + BN) / (8 * LW);
  static_assert((BM + BN) % (8 * LW) == 0 && BM % 32 == 0 && BN % 32 == 0 && NB >= 2 && (NB - 2) * PW < 64, "whole loads, and a count that vmcnt holds");
  using Acc = typename Op::Acc;

  // Whether this wavefront has outputs.
  __device__ static __forceinline__ bool run(const NtOperands& p, uint8_t* lds, int m0, int n0, int k_lo, int k_hi, int wave, int lane,
                                             Acc (&acc)[TN][TM]) {
    auto stage_begins = [&]() __attribute__((always_inline)) {
      __builtin_amdgcn_sched_barrier(0);
      asm volatile("s_barrier" ::: "memory");
      __builtin_amdgcn_sched_barrier(0);
    };
    if (wave >= CW) {
      const int w = wave - CW;
      const __amdgpu_buffer_rsrc_t rsa = nt_rows(p.a, m0, p.lda, min(BM, p.M - m0), p.K), rsb = nt_rows(p.b, n0, p.ldb, min(BN, p.N - n0), p.K / p.turns);
      const int lc = ((lane & 7) ^ ((lane >> 3) & 7)) * 16;  // (a load's 8 rows begin at a multiple of 8)
      int off[PW];
#pragma unroll
      for (int i = 0; i < PW; ++i) {
        const int q = w * PW + i;
        off[i] = (q < BM / 8 ? (q * 8 + (lane >> 3)) * p.lda : (q * 8 - BM + (lane >> 3)) * p.ldb) + lc;
      }
      const int part = nt_part(p);
      auto ask = [&](int t, int buf) __attribute__((always_inline)) {
        // past K, and past the last stage: zeros, and no memory is read
        const bool in = t < k_hi && t * 128 + lc < p.K;
        const int tb = nt_stage_of_b(t, part);
#pragma unroll
        for (int i = 0; i < PW; ++i) {
          const bool a = w * PW + i < BM / 8;
          nt_lds_load16(a ? rsa : rsb, lds + buf * STAGE + (w * PW + i) * 1024, in ? off[i] + (a ? t : tb) * 128 : kNtOutside);
        }
      };
      for (int t = 0; t < NB - 1; ++t) ask(k_lo + t, t);
      int buf = NB - 1;
      for (int t = k_lo; t < k_hi; ++t) {
        constexpr int left = (NB - 2) * PW;  // loads of later stages
        __builtin_amdgcn_s_waitcnt((left & 15) | (left >> 4) << 14 | 0x70 | 0xF00);
        stage_begins();
        ask(t + NB - 1, buf);  // the buffer of stage t - 1, which everyone has read
        buf = buf == NB - 1 ? 0 : buf + 1;
      }
      __builtin_amdgcn_s_waitcnt(0x70 | 0xF00);  // no load writes LDS after the block
      return false;
    }
#pragma unroll
    for (int i = 0; i < TN; ++i)
#pragma unroll
      for (int j = 0; j < TM; ++j) acc[i][j] = Acc{0, 0, 0, 0};
    const int lr = lane & 15, lk = lane >> 4;
    const uint32_t base = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint8_t*)lds + lr * 128 + (lk ^ (lr & 7)) * 16;
    const uint32_t at_a = base + wave / WN * WTM * 128, at_b = base + (BM + wave % WN * WTN) * 128;
    int buf = 0;
    for (int t = k_lo; t < k_hi; ++t) {
      stage_begins();
      i32x4 x[2][TM], y[2][TN];
      nt_read_stage<TM, TN>(at_a + buf * STAGE, at_b + buf * STAGE, x, y);
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int j = 0; j < TM; ++j)
#pragma unroll
          for (int i = 0; i < TN; ++i) acc[i][j] = Op::mma(y[h][i], x[h][j], acc[i][j]);
      buf = buf == NB - 1 ? 0 : buf + 1;
    }
    return true;
  }

  __device__ static __forceinline__ int row(int m0, int wave, int lane) { return m0 + wave / WN * WTM + (lane & 15); }
  __device__ static __forceinline__ int column(int n0, int wave, int lane) { return n0 + wave % WN * WTN + 4 * (lane >> 4); }
};

// The forms of tile, and what they take: us a stage of 128 bytes on a CU, with few CUs at work (alone) and with all (busy),
// fitted to timed calls of 48 to 4096 rows whose weights no cache holds (a traced launch alone is quicker: 333 x 4096 x 11008 on 192 CUs, 128 x 64,
// 86 stages of 0.35). A CU takes its blocks one after another or side by side; either
// way their stages add up. Bounds: what a CU's loads to LDS bring (86 to 91 bytes a ns; 64 x 64 reads four times as
// much a product as 256 x 256), a barrier a stage, and at 256 x 256 the matrix cores at the clock that they leave themselves.
struct NtForm {
  int bm, bn;
  float alone, busy;
};
inline constexpr NtForm kNtForms[] = {{64, 64, 0.24f, 0.23f}, {128, 64, 0.36f, 0.45f}, {128, 128, 0.52f, 0.60f}, {128, 128, 0.55f, 0.55f}, {256, 256, 1.35f, 1.85f}};

// The quickest form and number of ranges of K (bytes) by these figures: 4 us for a launch and its first stage; ranges cost a
// second launch and their sums' way through memory. Int8, us of each form (64 x 64, 128 x 64, 128 x 128, that in phases, 256 x 256; best
// in ranges): 333 x 4096 x 11008 43, 36, 49, 89, 133; 35 in two of 128 x 128. 1024 x 4096 x 4096 27, 26, 20, 29, 43.
// 2048 x 4096 x 4096 52, 50, 39, 38, 44. 4096 x 11008 x 4096 305, 339, 242, 238, 168. 64 x 4096 x 11008 31; 17 in four.
inline void nt_choose(int64_t M, int64_t N, int64_t K, int& form, int& splits) {
  const int64_t units = cdiv(K, 128);
  float best = 3e38f;
  for (int f = 0; f < 5; ++f) {
    const NtForm& t = kNtForms[f];
    const int64_t tiles = cdiv(M, t.bm) * cdiv(N, t.bn);
    for (int s = 1; s <= (f < 3 && M <= 65535 ? 8 : 1) && (s == 1 || units / s >= 4); ++s) {  // (the join has a block row a row)
      // (128 x 128 in phases needs two blocks a CU, which begin and end together)
      const int64_t deep = f == 3 ? 2 * cdiv(tiles, 512) : cdiv(tiles * s, 256);
      const float stage = deep > 1 ? t.busy : t.alone + (t.busy - t.alone) * (float)(tiles * s) / 256.0f;
      const float us = 4.0f + (float)(deep * cdiv(units, s)) * stage +
                       (s > 1 ? 8.0f + (float)s * (float)M * (float)N * 4.0f / 2.5e6f : 0.0f);
      if (us < best) {
        best = us;
        form = f;
        splits = s;
      }
    }
  }
}

// Calls f with the chosen form's type as Form<T>{}; those past the third take no ranges.
template <class T>
struct Form {
  using type = T;
};
template <class Op, class F>
int nt_form(int form, F f) {
  switch (form) {
    case 0: return f(Form<NtSmall<Op, 64, 64, 5, 4, 4>>{});
    case 1: return f(Form<NtSmall<Op, 128, 64, 6, 4, 4>>{});
    case 2: return f(Form<NtSmall<Op, 128, 128, 4, 8, 4>>{});
    case 3: return f(Form<NtTile<Op, 128, 2>>{});
    default: return f(Form<NtTile<Op, 256, 2>>{});
  }
}

}  // namespace mls
