// A tile of a product of two matrices whose rows both run along the reduction axis: 128 bytes of every row a
// stage, brought into LDS by loads that write it directly, two buffers, one barrier a stage.
//
// Op: the matrix instruction of 16 rows by 16 rows over 64 bytes of each (int8: 64 values, 16-bit types: 32):
// Acc and mma(first, second, acc). Lane (lr, lk) = (lane & 15, lane >> 4) gives row lr's 16-byte chunk lk of both and
// ends with the products of second's row lr and first's rows 4 lk .. 4 lk + 3.
//
// LDS: row r's chunk c lies in slot r * 8 + (c ^ (r & 7)), so that the 16 rows of an operand read, and the 8
// lanes that fill a row, cover all banks. The LDS-direct loads write lane l's chunk to slot base + l: each lane loads
// the chunk that belongs there.
#pragma once

#include "common.h"

namespace mls {

constexpr int kNtOutside = (int)0x80000000u;  // past every descriptor (they span < 2^31 bytes)

struct NtOperands {
  const uint8_t* a;  // [M][lda] bytes
  const uint8_t* b;  // [N][ldb]
  int lda, ldb;      // bytes, multiples of 16, as a and b
  int M, N, K;       // K: bytes of a row, a multiple of 16
};

// The rows first .. first + rows of a matrix. The offsets that lanes give are checked against it.
__device__ __forceinline__ __amdgpu_buffer_rsrc_t nt_rows(const void* base, int64_t first, int64_t ld, int rows, int K) {
  return __builtin_amdgcn_make_buffer_rsrc((void*)((const uint8_t*)base + first * ld), (short)0, (int)((rows - 1) * ld + K),
                                           0x00020000);
}

__device__ __forceinline__ void nt_lds_load16(__amdgpu_buffer_rsrc_t rs, void* lds, int voff) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (__attribute__((address_space(3))) void*)lds, 16, voff, 0, 0, 0);
}

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

template <class Op, int BM, int BN, int WM, int WN>
struct NtTile {
  static constexpr int NW = WM * WN, WTM = BM / WM, WTN = BN / WN, TM = WTM / 16, TN = WTN / 16;
  static constexpr int PA = BM * 8 / (64 * NW), PB = BN * 8 / (64 * NW);  // chunks a lane and stage
  static_assert(PA >= 1 && PB >= 1 && BM * 8 % (64 * NW) == 0 && BN * 8 % (64 * NW) == 0, "whole loads");
  using Acc = typename Op::Acc;

  // Stages k_lo .. k_hi of 128 bytes of the tile at (m0, n0). acc[i][j]: b's rows wn0 + 16 i .., a's 16 j ..
  __device__ static __forceinline__ void run(const NtOperands& p, int m0, int n0, int k_lo, int k_hi, int wave, int lane,
                                             Acc (&acc)[TN][TM]) {
    // separate arrays: the loads into one pair are known not to touch the pair being read
    __shared__ __align__(16) uint4 A0[BM * 8], B0[BN * 8], A1[BM * 8], B1[BN * 8];
    const int wm0 = (wave / WN) * WTM, wn0 = (wave % WN) * WTN;
    const __amdgpu_buffer_rsrc_t rsa = nt_rows(p.a, m0, p.lda, min(BM, p.M - m0), p.K);
    const __amdgpu_buffer_rsrc_t rsb = nt_rows(p.b, n0, p.ldb, min(BN, p.N - n0), p.K);
    const int lc = (lane & 7) ^ ((lane >> 3) & 7);
    int a_off[PA], b_off[PB];
#pragma unroll
    for (int i = 0; i < PA; ++i) a_off[i] = ((i * NW + wave) * 8 + (lane >> 3)) * p.lda + lc * 16;
#pragma unroll
    for (int i = 0; i < PB; ++i) b_off[i] = ((i * NW + wave) * 8 + (lane >> 3)) * p.ldb + lc * 16;
    auto dma = [&](uint4* as, uint4* bs, int kt) __attribute__((always_inline)) {
      const int k0 = kt * 128;
      // past K: a reads zeros, and b whatever its next row holds
      const bool in = k0 + lc * 16 < p.K;
#pragma unroll
      for (int i = 0; i < PA; ++i) nt_lds_load16(rsa, as + (i * NW + wave) * 64, in ? a_off[i] + k0 : kNtOutside);
#pragma unroll
      for (int i = 0; i < PB; ++i) nt_lds_load16(rsb, bs + (i * NW + wave) * 64, in || !Op::kZeroB ? b_off[i] + k0 : kNtOutside);
    };
#pragma unroll
    for (int i = 0; i < TN; ++i)
#pragma unroll
      for (int j = 0; j < TM; ++j) acc[i][j] = Acc{0, 0, 0, 0};

    const int lr = lane & 15, lk = lane >> 4;
    // Stage kt lies in one pair of buffers; at its start the loads of stage kt + 1 go into the other pair,
    // last read before the barrier that ended stage kt - 1. The closing wait covers them.
    auto stage = [&](const uint4* as, const uint4* bs, uint4* an, uint4* bn, int kt) __attribute__((always_inline)) {
      __builtin_amdgcn_sched_barrier(0);
      if (kt + 1 < k_hi) dma(an, bn, kt + 1);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        uint4 bop[TN];
#pragma unroll
        for (int i = 0; i < TN; ++i) {
          const int row = wn0 + i * 16 + lr;
          bop[i] = bs[row * 8 + ((lk + 4 * h) ^ (row & 7))];
        }
#pragma unroll
        for (int j = 0; j < TM; ++j) {
          const int row = wm0 + j * 16 + lr;
          const uint4 aop = as[row * 8 + ((lk + 4 * h) ^ (row & 7))];
#pragma unroll
          for (int i = 0; i < TN; ++i) acc[i][j] = Op::mma(bop[i], aop, acc[i][j]);
        }
      }
      __builtin_amdgcn_sched_barrier(0);
      asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
      __builtin_amdgcn_sched_barrier(0);
    };
    if (k_lo < k_hi) dma(A0, B0, k_lo);
    __syncthreads();
    int kt = k_lo;
    for (; kt + 2 <= k_hi; kt += 2) {
      stage(A0, B0, A1, B1, kt);
      stage(A1, B1, A0, B0, kt + 1);
    }
    if (kt < k_hi) stage(A0, B0, A1, B1, kt);
  }

  // f(m, n, acc): the outputs (m, n .. n + 3) of this lane, m < M, n < N
  template <class F>
  __device__ static __forceinline__ void each(const NtOperands& p, int m0, int n0, int wave, int lane, const Acc (&acc)[TN][TM], F f) {
    const int mb = m0 + (wave / WN) * WTM + (lane & 15), nb = n0 + (wave % WN) * WTN + 4 * (lane >> 4);
#pragma unroll
    for (int i = 0; i < TN; ++i)
#pragma unroll
      for (int j = 0; j < TM; ++j)
        if (mb + 16 * j < p.M && nb + 16 * i < p.N) f(mb + 16 * j, nb + 16 * i, acc[i][j]);
  }
};

}  // namespace mls
