// 8-bit codes of activations: the scale of a group of values, and the codes under it.
//
// scale = max(amax / 127, 1e-8), code = x / scale rounded to the nearest whole number, ties to even:
// what the weights' quantizers do (quant.hip), bit for bit, with one division a group instead of one a
// value.
#pragma once

#include "common.h"

namespace mls {

// |x| as bits: unsigned comparison orders them as numbers, infinity above them and NaN above that, so a
// maximum over bits keeps a NaN (which fmaxf drops).
__device__ __forceinline__ uint32_t abs_bits(float x) { return __float_as_uint(x) & 0x7FFFFFFFu; }

template <int C>
struct Dpp {
  static constexpr int v = C;
};

struct Scale8 {
  float s, inv;
  uint32_t finite;  // all bits, or none: the codes under an infinite or NaN scale are 0
};

// inv: 1 / s, rounded to nearest
__device__ __forceinline__ Scale8 scale8(uint32_t amax_bits) {
  float s = __uint_as_float(amax_bits) / 127.0f;
  if (s < 1e-8f) s = 1e-8f;  // (a NaN stays)
  return {s, 1.0f / s, amax_bits < 0x7F800000u ? ~0u : 0u};
}

// A float whose low byte is the code of x. t is within one ulp of x / s, and where inv is 1 / s rounded to
// nearest, t plus its remainder times inv, rounded once, is x / s rounded to nearest (Markstein's
// division): four operations instead of a division's ten. Adding 1.5 * 2^23 rounds that to a whole number, ties to even,
// held in the low bits as two's complement. |x| / s is at most 127 (1 + 2^-24), so no code is past 127.
__device__ __forceinline__ uint32_t code8(float x, const Scale8& g) {
  const float t = x * g.inv;
  const float q = fmaf(fmaf(-t, g.s, x), g.inv, t);
  return __float_as_uint(q + 12582912.0f);
}

__device__ __forceinline__ uint32_t pack_codes(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  const uint32_t lo = __builtin_amdgcn_perm(b, a, 0x0C0C0400u), hi = __builtin_amdgcn_perm(d, c, 0x0C0C0400u);
  return lo | (hi << 16);
}

__device__ __forceinline__ uint2 codes8(const float (&v)[8], const Scale8& g) {
  return make_uint2(pack_codes(code8(v[0], g), code8(v[1], g), code8(v[2], g), code8(v[3], g)) & g.finite,
                    pack_codes(code8(v[4], g), code8(v[5], g), code8(v[6], g), code8(v[7], g)) & g.finite);
}

// 8 consecutive values of a row as they lie there, of a K that is a multiple of 8 (past K: others of the row). Without a
// branch, so that several are on their way at once: a load8 is waited for within its own.
template <typename T>
struct Raw8 {
  T v[8];
};
template <typename T>
__device__ __forceinline__ Raw8<T> fetch8(const T* row, int64_t k, int64_t K) {
  Raw8<T> r;
  const int64_t other = (threadIdx.x & 63) * 8;
  __builtin_memcpy(&r, row + (k < K ? k : other < K ? other : 0), sizeof(r));
  return r;
}
template <typename T>
__device__ __forceinline__ void widen8(const Raw8<T>& r, bool in, float (&v)[8]) {
#pragma unroll
  for (int e = 0; e < 8; ++e) v[e] = in ? to_f32(r.v[e]) : 0.0f;
}

// 8 consecutive values of a row from column k, zeros past K; any alignment of a whole number of values.
template <typename T>
__device__ __forceinline__ void load8(const T* row, int64_t k, int64_t K, float (&v)[8]) {
  if (k + 8 <= K) {
    T raw[8];
    __builtin_memcpy(raw, row + k, sizeof(raw));
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = to_f32(raw[e]);
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = k + e < K ? to_f32(row[k + e]) : 0.0f;
  }
}

__device__ __forceinline__ void codes_to_values(uint32_t lo, uint32_t hi, float s, float (&v)[8]) {
#pragma unroll
  for (int e = 0; e < 8; ++e) v[e] = (float)(int8_t)((e < 4 ? lo : hi) >> (8 * (e % 4))) * s;
}

// 8 consecutive codes of a row from column k as values, zeros past K; any alignment.
__device__ __forceinline__ void load_codes8(const int8_t* row, int64_t k, int64_t K, float s, float (&v)[8]) {
  uint32_t w[2] = {0, 0};
  if (k + 8 <= K) {
    __builtin_memcpy(w, row + k, 8);
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (k + e < K) w[e / 4] |= (uint32_t)(uint8_t)row[k + e] << (8 * (e % 4));
  }
  codes_to_values(w[0], w[1], s, v);
}

// n <= 8 values to a row; any alignment of a whole number of values.
template <typename T>
__device__ __forceinline__ void store8(T* dst, const float (&v)[8], int64_t n) {
  T raw[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) raw[e] = from_f32<T>(v[e]);
  if (n >= 8) {
    __builtin_memcpy(dst, raw, sizeof(raw));
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (e < n) dst[e] = raw[e];
  }
}

__device__ __forceinline__ uint32_t max_abs8(const float (&v)[8]) {
  uint32_t m = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e) m = max(m, abs_bits(v[e]));
  return m;
}

// Maximum over each aligned group of W >= 16 lanes, in all of them.
template <int W>
__device__ __forceinline__ uint32_t group_max_bits(uint32_t v) {
  static_assert(W == 16 || W == 64, "a DPP row, or the wavefront");
  auto dpp = [&](auto ctrl) __attribute__((always_inline)) {
    v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, decltype(ctrl)::v, 0xF, 0xF, false));
  };
  dpp(Dpp<0xB1>{});   // lane ^ 1
  dpp(Dpp<0x4E>{});   // lane ^ 2
  dpp(Dpp<0x141>{});  // the other quad of the octet
  dpp(Dpp<0x140>{});  // the other octet
  if constexpr (W == 64) {
    v = max(v, (uint32_t)__shfl_xor((int)v, 16, 64));
    v = max(v, (uint32_t)__shfl_xor((int)v, 32, 64));
  }
  return v;
}

// silu'(g) and silu(g) need sig = 1 / (1 + e^-g). For 16-bit values the hardware's exponential and
// reciprocal (a few 2^-23 off) are far below their rounding; fp32 takes the exact forms.
template <typename T>
__device__ __forceinline__ float sigmoid(float g) {
  if constexpr (sizeof(T) == 4) return 1.0f / (1.0f + expf(-g));
  return __builtin_amdgcn_rcpf(1.0f + __expf(-g));
}

constexpr int kGroup8 = 128;  // columns that share a scale in a checkpoint

// act8.hip: codes [M][ldq] (zeros in columns K .. kpad) and scales [M] of x's rows
int launch_quantize_rows(const void* x, int dt, int64_t ldx, int64_t M, int64_t K, int64_t kpad, int8_t* q,
                         int64_t ldq, float* s, hipStream_t st);
// bytes src [rows][ld] -> dst [rows][kpad], kpad a multiple of 16, zeros from column K, of two matrices in one launch
struct PadRows {
  const uint8_t* src;
  int64_t ld, rows;
  uint8_t* dst;
};
// Whether a launch stays below 2^32 threads, the most that a grid has.
inline bool grid_fits(int64_t blocks, int64_t threads) { return blocks <= 0xFFFFFFFFll / threads; }

int launch_pad_rows(const PadRows& one, const PadRows& two, int64_t K, int64_t kpad, hipStream_t st);

}  // namespace mls
