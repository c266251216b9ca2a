// New keys and values into a paged cache, rotated by position on the way, and the queries
// rotated beside them: one launch between the q/k/v projections and the attention that reads the
// cache. A pair (a, b) at position p, angle j: (a cos - b sin, a sin + b cos), in fp32, rounded once.
//
// HBM-bound: q, k, v and the rotation table's rows are read once, q', K and V written once. One
// wavefront per (row, part of its heads); a lane keeps one place of a head (16 bytes, or the two
// 16-byte halves that hold its pairs) over all of the wavefront's heads, so the cosines and
// sines are loaded once. Rows are cut into parts only until the GPU is filled. 10.7K tokens of 32 + 2 x 8 heads of 128, bf16
// (267 MB): 50 us, 5.3 TB/s; 64 tokens 3.8 us, a launch.
#include <algorithm>

#include "paged_gqa_args.h"

namespace mls {

namespace {

struct AppendArgs {
  const void *q, *k, *v;
  void *kp, *vp, *qo;
  const int32_t *bt, *lens, *cu;
  const float* rope;
  int64_t q_st, q_sh, k_st, k_sh, v_st, v_sh, kv_sb, kv_sh, kv_st, bt_ss, rope_ld, num_blocks;
  int n, T, Hq, Hkv, D, BS, max_blocks, rope_rows, rot, parts;
};

// U elements of T in one access (U = 16 / sizeof(T)), or element by element up to `left` of them
template <typename T, int U, bool VEC>
__device__ __forceinline__ void load_u(const T* p, int left, float (&x)[U]) {
  if constexpr (VEC) {
    const uint4 v = *reinterpret_cast<const uint4*>(p);
    const T* h = reinterpret_cast<const T*>(&v);
#pragma unroll
    for (int i = 0; i < U; ++i) x[i] = to_f32(h[i]);
  } else {
#pragma unroll
    for (int i = 0; i < U; ++i) x[i] = i < left ? to_f32(p[i]) : 0.0f;
  }
}
template <typename T, int U, bool VEC>
__device__ __forceinline__ void store_u(T* p, int left, const float (&x)[U]) {
  if constexpr (VEC) {
    T h[U];
#pragma unroll
    for (int i = 0; i < U; ++i) h[i] = from_f32<T>(x[i]);
    *reinterpret_cast<uint4*>(p) = __builtin_bit_cast(uint4, h);
  } else {
#pragma unroll
    for (int i = 0; i < U; ++i)
      if (i < left) p[i] = from_f32<T>(x[i]);
  }
}

// A place of a head: U elements at d; half-split pairs (IL = false): U more at d + rot / 2.
template <typename T, int U, bool VEC, bool IL>
__global__ __launch_bounds__(256) void paged_append_kernel(const AppendArgs a) {
  const int lane = threadIdx.x & 63;
  const int64_t item = (int64_t)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (item >= (int64_t)a.T * a.parts) return;
  const int tok = (int)(item / a.parts), part = (int)(item % a.parts);
  int seq = tok, pos;
  bool real = true;
  if (a.cu) {
    auto start = [&](int s) { return min(max(a.cu[s], 0), a.T); };
    seq = __builtin_amdgcn_readfirstlane(last_start(a.n, tok, lane, start));
    real = seq >= 0 && seq < a.n;
    pos = real ? a.lens[seq] - (start(seq + 1) - tok) : -1;
  } else {
    pos = a.lens[seq] - 1;
  }
  int64_t slot = -1;  // elements into the pools
  if (real && pos >= 0 && pos / a.BS < a.max_blocks) {
    const int blk = a.bt[seq * a.bt_ss + pos / a.BS];
    if (blk >= 0 && blk < a.num_blocks) slot = blk * a.kv_sb + (int64_t)(pos % a.BS) * a.kv_st;
  }
  const int half = a.rot / 2;
  const int turned = a.rope ? (IL ? a.rot : half) / U : 0;        // places with pairs
  const int from = a.rope ? a.rot : 0;                            // first element without
  const int places = turned + (a.D - from + U - 1) / U;
  // the q and k heads; places wider than a wavefront take several rounds
  const int width = min(places, 64), per = 64 / width, hl = lane / width;
  const int Hr = (a.rope && a.q ? a.Hq : 0) + a.Hkv, k0 = Hr - a.Hkv;
  for (int c = lane % width; c < places && hl < per; c += width) {
    const bool turn = c < turned;
    const int d = turn ? c * U : from + (c - turned) * U, left = a.D - d;
    float cs[U], sn[U];
    if (turn) {
      const bool in = pos >= 0 && pos < a.rope_rows;
      const float* r = a.rope + (in ? (int64_t)pos * a.rope_ld : 0);
#pragma unroll
      for (int i = 0; i < U; ++i) {
        const int j = IL ? (d + i) / 2 : d + i;
        cs[i] = in ? r[j] : __builtin_nanf("");
        sn[i] = in ? r[half + j] : __builtin_nanf("");
      }
    }
    for (int h = part * per + hl; h < Hr; h += per * a.parts) {
      const bool isq = h < k0;
      const T* src = isq ? static_cast<const T*>(a.q) + tok * a.q_st + h * a.q_sh
                         : static_cast<const T*>(a.k) + tok * a.k_st + (h - k0) * a.k_sh;
      T* dst = isq ? static_cast<T*>(a.qo) + ((int64_t)tok * a.Hq + h) * a.D
                   : static_cast<T*>(a.kp) + slot + (h - k0) * a.kv_sh;
      if (!isq && slot < 0) continue;
      float x[U];
      load_u<T, U, VEC>(src + d, left, x);
      if (!turn) {
        if (isq && !real)
#pragma unroll
          for (int i = 0; i < U; ++i) x[i] = 0.0f;
        store_u<T, U, VEC>(dst + d, left, x);
        continue;
      }
      float y[U];
      if constexpr (IL) {
#pragma unroll
        for (int i = 0; i < U; i += 2) {
          y[i] = x[i] * cs[i] - x[i + 1] * sn[i];
          y[i + 1] = x[i] * sn[i] + x[i + 1] * cs[i];
        }
        if (isq && !real)
#pragma unroll
          for (int i = 0; i < U; ++i) y[i] = 0.0f;
        store_u<T, U, VEC>(dst + d, left, y);
      } else {
        float z[U], w[U];
        load_u<T, U, VEC>(src + d + half, left, z);
#pragma unroll
        for (int i = 0; i < U; ++i) {
          y[i] = x[i] * cs[i] - z[i] * sn[i];
          w[i] = x[i] * sn[i] + z[i] * cs[i];
          if (isq && !real) y[i] = w[i] = 0.0f;
        }
        store_u<T, U, VEC>(dst + d, left, y);
        store_u<T, U, VEC>(dst + d + half, left, w);
      }
    }
  }
  // v, as it is
  if (slot < 0) return;
  const int vplaces = (a.D + U - 1) / U;
  for (int e = part * 64 + lane; e < vplaces * a.Hkv; e += 64 * a.parts) {
    const int h = e / vplaces, d = (e % vplaces) * U;
    const T* src = static_cast<const T*>(a.v) + tok * a.v_st + h * a.v_sh + d;
    T* dst = static_cast<T*>(a.vp) + slot + h * a.kv_sh + d;
    if constexpr (VEC) {
      *reinterpret_cast<uint4*>(dst) = *reinterpret_cast<const uint4*>(src);
    } else {
#pragma unroll
      for (int i = 0; i < U; ++i)
        if (d + i < a.D) dst[i] = src[i];
    }
  }
}

template <typename T>
int launch_append(const AppendArgs& a, bool vec, bool il, hipStream_t st) {
  constexpr int CE = 16 / (int)sizeof(T);
  const dim3 grid((unsigned)cdiv((int64_t)a.T * a.parts, 4)), block(256);
  if (vec && il) hipLaunchKernelGGL((paged_append_kernel<T, CE, true, true>), grid, block, 0, st, a);
  else if (vec) hipLaunchKernelGGL((paged_append_kernel<T, CE, true, false>), grid, block, 0, st, a);
  else if (il) hipLaunchKernelGGL((paged_append_kernel<T, 2, false, true>), grid, block, 0, st, a);
  else hipLaunchKernelGGL((paged_append_kernel<T, 1, false, false>), grid, block, 0, st, a);
  return check_launch("mlsx_paged_append");
}

}  // namespace

}  // namespace mls

using namespace mls;

extern "C" int mlsx_paged_append(const mlsx_paged_append_args* p, mls_stream_t stream) {
  const char* fn = "mlsx_paged_append";
  if (!p) return fail(MLS_ERR_ARG, "%s: null arguments", fn);
  if (p->n_seqs < 0 || p->tokens < 0 || p->heads < 0 || p->kv_heads < 0 || p->head_dim < 0 || p->block_size < 1 ||
      p->max_blocks < 0 || p->num_blocks < 0 || p->rope_rows < 0)
    return fail(MLS_ERR_ARG, "%s: bad sizes n_seqs=%lld tokens=%lld heads=%lld kv_heads=%lld head_dim=%lld block_size=%lld", fn,
                (long long)p->n_seqs, (long long)p->tokens, (long long)p->heads, (long long)p->kv_heads, (long long)p->head_dim,
                (long long)p->block_size);
  if (p->dt != MLS_F32 && p->dt != MLS_F16 && p->dt != MLS_BF16) return fail(MLS_ERR_ARG, "%s: bad dtype", fn);
  const bool queries = p->q && p->rope && p->rot > 0 && p->heads > 0;
  if (p->tokens == 0 || p->head_dim == 0 || (p->kv_heads == 0 && !queries)) return MLS_OK;
  if ((p->kv_heads > 0 && (!p->k || !p->v || !p->k_pool || !p->v_pool)) || (queries && !p->q_out) ||
      (p->n_seqs > 0 && (!p->context_lens || (p->max_blocks > 0 && !p->block_tables))))
    return fail(MLS_ERR_ARG, "%s: null pointer", fn);
  if (!p->cu_seqlens && p->tokens != p->n_seqs)
    return fail(MLS_ERR_ARG, "%s: %lld rows for %lld sequences of one", fn, (long long)p->tokens, (long long)p->n_seqs);
  if (!p->rope && p->rot > 0) return fail(MLS_ERR_ARG, "%s: %lld rotated elements without a table", fn, (long long)p->rot);
  if (p->rope && (p->rot < 0 || p->rot % 2 != 0 || p->rot > p->head_dim || p->rope_ld < p->rot))
    return fail(MLS_ERR_ARG, "%s: %lld rotated elements of %lld, table rows of %lld", fn, (long long)p->rot,
                (long long)p->head_dim, (long long)p->rope_ld);
  if (p->kv_st < p->head_dim || p->kv_sh < p->head_dim || p->kv_sb < 0 || p->q_st < 0 || p->q_sh < 0 || p->k_st < 0 ||
      p->k_sh < 0 || p->v_st < 0 || p->v_sh < 0 || p->bt_ss < 0)
    return fail(MLS_ERR_ARG, "%s: bad strides", fn);
  if (p->tokens > 0x3FFFFFFF || p->n_seqs > 0x3FFFFFFF || p->heads > 65535 || p->kv_heads > 65535 || p->head_dim > 65536 ||
      p->block_size > 0x3FFFFFFF || p->max_blocks > 0x7FFFFFFF || p->rope_rows > 0x7FFFFFFF)
    return fail(MLS_ERR_UNSUPPORTED, "%s: too large", fn);
  AppendArgs a{p->q, p->k, p->v, p->k_pool, p->v_pool, p->q_out, p->block_tables, p->context_lens, p->cu_seqlens,
               p->rot > 0 ? p->rope : nullptr, p->q_st, p->q_sh, p->k_st, p->k_sh, p->v_st, p->v_sh, p->kv_sb, p->kv_sh,
               p->kv_st, p->bt_ss, p->rope_ld, p->num_blocks, (int)p->n_seqs, (int)p->tokens, (int)p->heads, (int)p->kv_heads,
               (int)p->head_dim, (int)p->block_size, (int)p->max_blocks, (int)p->rope_rows, p->rope ? (int)p->rot : 0, 1};
  const int esz = dt_size(p->dt), ce = 16 / esz;
  const bool il = p->interleaved != 0;
  auto whole = [&](int64_t v) { return v % ce == 0; };
  const bool vec = whole(a.D) && whole(il ? a.rot : a.rot / 2) && whole(a.k_st) && whole(a.k_sh) && whole(a.v_st) &&
                   whole(a.v_sh) && whole(a.kv_sb) && whole(a.kv_sh) && whole(a.kv_st) && aligned(a.k, 16) && aligned(a.v, 16) &&
                   aligned(a.kp, 16) && aligned(a.vp, 16) &&
                   (!queries || (whole(a.q_st) && whole(a.q_sh) && aligned(a.q, 16) && aligned(a.qo, 16)));
  // parts: the rounds that a row's heads take, as far as the GPU has room
  const int u = vec ? ce : il ? 2 : 1;
  const int places = a.rot / u / (il ? 1 : 2) + (int)cdiv(a.D - a.rot, u);
  const int64_t heads = (queries ? a.Hq : 0) + a.Hkv, rounds = cdiv(heads, 64 / std::min(std::max(places, 1), 64));
  a.parts = (int)std::max<int64_t>(1, std::min(rounds, cdiv(4096, a.T)));
  if (cdiv((int64_t)a.T * a.parts, 4) > 0x7FFFFFFF) return fail(MLS_ERR_UNSUPPORTED, "%s: too large", fn);
  if (!queries) a.q = nullptr;
  hipStream_t st = (hipStream_t)stream;
  if (p->dt == MLS_F32) return launch_append<float>(a, vec, il, st);
  if (p->dt == MLS_F16) return launch_append<_Float16>(a, vec, il, st);
  return launch_append<__bf16>(a, vec, il, st);
}
