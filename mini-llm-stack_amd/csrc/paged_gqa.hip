// Attention over a paged K/V cache for prompts, chunks, drafted and single tokens, with grouped
// heads, score caps, biases by distance, windows and prefix masks, and for batches behind one
// shared prefix: host side and the join of pieces. The kernels are in paged_gqa.h.
//
// Row i of a sequence (position p, K/V head h) sees key j < len when j <= p or j < prefix, and,
// with a window w, p - j < w. Its score is x = scale q.k, capped c tanh(x / c), less
// slope |p - j|; out = sum_j softmax(x)_j v_j, 0 where it sees nothing.
//
// Three kernels:
// - gqa_keys_kernel, up to 16 packed rows (new tokens x group) a sequence: HBM-bound. Each
//   wavefront streams keys of its own, all hold the same rows.
// - gqa_pair_kernel, many rows of 16-bit types: MFMA-bound. 8 wavefronts of 32 rows (16 of D > 128) share the K/V
//   tiles, in two groups of which one multiplies while the other makes its softmax.
// - gqa_rows_kernel, the rest (fp32, rows between, any alignment): 4 wavefronts of 16 or 32 rows share the tiles.
// Where row tiles are fewer than the GPU has room for, contexts are cut into pieces, whose
// (O, reference, sum) a fourth kernel joins. A shared prefix is a pass of its own: the rows of all
// sequences against its keys, read once for a tile of rows instead of once a sequence.
#include <algorithm>

#include "paged_gqa_args.h"

namespace mls {

template <typename T> int gqa_launch(const GqaArgs& a, const GqaShape& s, int64_t blocks, hipStream_t st);
template <typename T> void gqa_tiles(GqaShape& s);
extern template int gqa_launch<float>(const GqaArgs&, const GqaShape&, int64_t, hipStream_t);
extern template int gqa_launch<_Float16>(const GqaArgs&, const GqaShape&, int64_t, hipStream_t);
extern template int gqa_launch<__bf16>(const GqaArgs&, const GqaShape&, int64_t, hipStream_t);
extern template void gqa_tiles<float>(GqaShape&);
extern template void gqa_tiles<_Float16>(GqaShape&);

namespace {

// One wavefront per (row, head): lane i holds piece i's reference and sum (at most 64 pieces); then DW / 4
// lanes take a record, 4 floats each, as many records at once as the wavefront has lanes for, four
// such loads in flight.
template <typename T>
__global__ __launch_bounds__(256) void gqa_join_kernel(const GqaArgs a) {
  const int lane = threadIdx.x & 63;
  const int Hq = a.Hkv * a.group;
  const int64_t item = (int64_t)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (item >= (int64_t)a.T * Hq) return;
  // (where offsets do not rise, no tile may have held the row: its count is whatever the workspace held)
  const int live = a.piece0 + min(max(__builtin_amdgcn_readfirstlane(a.ws_live[item]), 1), a.pieces - a.piece0);
  const float2* ml = reinterpret_cast<const float2*>(a.ws_ml) + item * a.pieces;
  const float2 x = ml[min(lane, live - 1)];
  if (live == 1) return;  // written by its only piece
  const float m = lane < live ? x.x : -3.402823466e38f;
  const float M = wave_max(m);
  const float f = lane < live ? __builtin_amdgcn_exp2f(m - M) : 0.0f;
  const float L = lane_group_sum<64>(lane < live ? x.y * f : 0.0f);
  const float g = L == 0.0f ? 0.0f : f / L;
  const int lanes = a.DW / 4, per = 64 / lanes, sub = lane / lanes, d = (lane % lanes) * 4;
  const float* w = a.ws + item * a.pieces * a.DW + d;
  f32x4 acc{0.f, 0.f, 0.f, 0.f};
  for (int s0 = 0; s0 < live; s0 += 4 * per) {
    f32x4 v[4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
      v[i] = *reinterpret_cast<const f32x4*>(w + (int64_t)min(s0 + i * per + sub, live - 1) * a.DW);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int s = s0 + i * per + sub;
      const float h = __shfl(g, min(s, 63), 64);
      if (s < live && sub < per) acc += v[i] * h;
    }
  }
  f32x4 sum = acc;
  for (int k = 1; k < per; ++k)
#pragma unroll
    for (int i = 0; i < 4; ++i) sum[i] += __shfl(acc[i], lane + k * lanes, 64);
  if (sub != 0) return;
  T* op = static_cast<T*>(a.out) + (item / Hq) * a.o_st + (item % Hq) * a.o_sh + d;
  if (a.o_vec && d + 4 <= a.D) {
    store4<T>(op, sum[0], sum[1], sum[2], sum[3]);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (d + i < a.D) op[i] = from_f32<T>(sum[i]);
  }
}

template <typename T>
int launch_join(const GqaArgs& a, hipStream_t st) {
  hipLaunchKernelGGL((gqa_join_kernel<T>), dim3((unsigned)cdiv((int64_t)a.T * a.Hkv * a.group, 4)), dim3(256), 0, st, a);
  return check_launch("paged attention (join)");
}

struct Pass {
  GqaArgs a;
  GqaShape s;
  int64_t blocks;
};

// Row tile and kernel for `rows` packed rows a sequence, `all` of them over all sequences and K/V heads.
// - Up to 16 rows: the kernel over keys (40 sequences of 1 to 4096 tokens, 4 rows: 40 us, the next one 58). With 32 rows a
//   wavefront it is out of registers: 32 rows, 12 sequences of up to 2048, 40 us against 28; 64 of 2000 to 6000, 323
//   against 239 (20 rows: 230 against 241).
//   (Weights are rounded once from here on: in two parts, 36 rows of 12 sequences 30.0 us against 28.2, 20 of 64 257 against 241.)
// - 16-bit types: the paired kernel's tiles of 256 rows (128 of D > 128) where they are at least half full, since it is
//   1.7 times as fast a row as tiles of 64 (prompt of 8192: 550 us, 915 in tiles of 64; 12 sequences of 192 new rows
//   52 against 57; of 96 rows 47 in the paired kernel, 37 in tiles of 64).
// - fp32: tiles of 128 rows where there are enough to fill the GPU (a step of one takes 3.4 us: 5 prompts of up to 700 tokens, 8 heads of 64,
//   47 us so, 31 in tiles of 64).
void choose_shape(GqaShape& s, int64_t rows, int64_t all, int dt, int64_t D, int64_t BS, bool vec, bool tanh) {
  s.dp = D <= 64 ? 64 : D <= 96 ? 96 : D <= 128 ? 128 : 256;
  if (dt == MLS_F32) gqa_tiles<float>(s);
  else gqa_tiles<_Float16>(s);
  vec = vec && BS % s.group_rows == 0;
  s.vec = vec;
  s.keys = vec && rows <= 16;
  s.pair = vec && !s.keys && dt != MLS_F32 && !tanh && rows > (s.dp <= 128 ? 128 : 64);
  s.nt = dt == MLS_F32 && vec && rows > 64 && all >= 128 * 512 ? 2 : 1;
  if (dt == MLS_F32) gqa_tiles<float>(s);
  else gqa_tiles<_Float16>(s);
}

// Validates a call and lays out its launches; need: floats of workspace.
int prepare(const char* fn, const mlsx_paged_attention_args* p, float* ws, Pass& own, Pass& pre, bool& shared, int64_t& need) {
  need = 0;
  own.blocks = pre.blocks = 0;
  shared = p->prefix_blocks != nullptr;
  const int64_t n = p->n_seqs, T = p->tokens, Hkv = p->kv_heads, G = p->group, D = p->head_dim, BS = p->block_size;
  if (n < 0 || T < 0 || Hkv < 0 || G < 0 || D < 0 || BS < 1 || p->max_blocks < 0 || p->num_blocks < 0 || p->window < 0 ||
      p->prefix_len < 0 || p->max_new < 0)
    return fail(MLS_ERR_ARG, "%s: bad sizes n_seqs=%lld tokens=%lld kv_heads=%lld group=%lld head_dim=%lld block_size=%lld",
                fn, (long long)n, (long long)T, (long long)Hkv, (long long)G, (long long)D, (long long)BS);
  if (p->dt != MLS_F32 && p->dt != MLS_F16 && p->dt != MLS_BF16) return fail(MLS_ERR_ARG, "%s: bad dtype", fn);
  if (T == 0 || Hkv == 0 || G == 0 || D == 0) return MLS_OK;
  if (!p->q || !p->k_pool || !p->v_pool || !p->out || (n > 0 && (!p->context_lens || (p->max_blocks > 0 && !p->block_tables))))
    return fail(MLS_ERR_ARG, "%s: null pointer", fn);
  if (!p->cu_seqlens && T != n) return fail(MLS_ERR_ARG, "%s: %lld rows for %lld sequences of one", fn, (long long)T, (long long)n);
  if (shared && p->cu_seqlens) return fail(MLS_ERR_ARG, "%s: a shared prefix takes one token a sequence", fn);
  if (p->q_sh < D || p->q_st < 0 || p->o_sh < D || p->o_st < Hkv * G * D || p->kv_sb < 0 || p->bt_ss < 0 ||
      (p->kv_st < D && p->kv_st != 0) || (p->kv_sh < D && p->kv_sh != 0))
    return fail(MLS_ERR_ARG, "%s: bad strides", fn);
  if (D > 256) return fail(MLS_ERR_UNSUPPORTED, "%s: head dim %lld above 256", fn, (long long)D);
  if (T * G > 0x3FFFFFFF || T * Hkv * G > 0x3FFFFFFFFll || n > 0x3FFFFFFF || BS > 0x3FFFFFFF || p->max_blocks > 0x7FFFFFFF ||
      p->window > 0x7FFFFFFF || p->prefix_len > 0x3FFFFFFF || Hkv > 65535 || G > 65535)
    return fail(MLS_ERR_UNSUPPORTED, "%s: too large", fn);
  if (!(p->softcap >= 0.0) || p->softcap > 3e38) return fail(MLS_ERR_ARG, "%s: softcap %g", fn, p->softcap);
  const int esz = dt_size(p->dt), ce = 16 / esz;
  const bool vec = D % ce == 0 && p->kv_st % ce == 0 && p->kv_sh % ce == 0 && p->kv_sb % ce == 0 && aligned(p->k_pool, 16) &&
                   aligned(p->v_pool, 16);
  GqaArgs a{};
  a.q = p->q, a.q_st = p->q_st, a.q_sh = p->q_sh;
  a.kp = p->k_pool, a.vp = p->v_pool, a.kv_sb = p->kv_sb, a.kv_sh = p->kv_sh, a.kv_st = p->kv_st;
  a.bt = p->block_tables, a.bt_ss = p->bt_ss, a.lens = p->context_lens, a.cu = p->cu_seqlens, a.prefix = p->prefix_lens;
  a.slopes = p->slopes, a.out = p->out, a.o_st = p->o_st, a.o_sh = p->o_sh;
  a.num_blocks = p->num_blocks, a.n = (int)n, a.T = (int)T, a.Hkv = (int)Hkv, a.group = (int)G, a.D = (int)D;
  a.DW = (int)cdiv(D, 4) * 4, a.BS = (int)BS;
  a.bs_magic = (uint32_t)((0xFFFFFFFFull / (uint64_t)BS) + 1);  // ceil(2^32 / BS) for BS > 1
  a.max_keys = (int)std::min<int64_t>(p->max_blocks * BS, 0x7FFFFFFF), a.window = (int)p->window;
  if (vec && p->kv_sb * esz <= 0xFFFFFFFFll && p->kv_st * esz * std::max<int64_t>(BS, 64) < 0x7FFFFFFFll)
    a.sb_bytes = (uint32_t)(p->kv_sb * esz), a.st_bytes = (uint32_t)(p->kv_st * esz);
  a.kv_vec = vec;
  constexpr double LOG2E = 1.4426950408889634;
  a.c = (float)(p->scale * LOG2E);
  // (a cap is none for scores under 2^-12 of it, in fp32; past 1e30, scale / cap and the cap leave fp32's normal values)
  const double cap = p->softcap <= 1e30 ? p->softcap : 0.0;
  a.cap = (float)(cap * LOG2E);
  a.to_cap = cap > 0.0 ? (float)std::clamp(p->scale / cap, -3e38, 3e38) : 0.0f;
  a.simple = a.cap == 0.0f && !a.slopes && a.c > 0.0f && a.c < 3e38f;
  a.q_vec = D % ce == 0 && p->q_st % ce == 0 && p->q_sh % ce == 0 && aligned(p->q, 16);
  a.o_vec = p->o_st % 4 == 0 && p->o_sh % 4 == 0 && aligned(p->out, 4 * esz);

  // the sequences' own keys
  own.a = a;
  own.s = pre.s = GqaShape{};
  const int64_t most = p->cu_seqlens ? (p->max_new > 0 ? std::min(p->max_new, T) : cdiv(T, std::max<int64_t>(n, 1))) : 1;
  choose_shape(own.s, most * G, T * G * Hkv, p->dt, D, BS, a.sb_bytes != 0, gqa_cap_needs_tanh(a));
  own.a.bm_log = __builtin_ctz(own.s.bm);
  own.a.bn_log = __builtin_ctz(own.s.bn);
  const int64_t bm = 1ll << own.a.bm_log;
  const int64_t slots = p->cu_seqlens ? T * G / bm + n + 2 : n * cdiv(G, bm);
  int64_t steps = cdiv(std::max<int64_t>(p->max_blocks * BS, 1), own.s.bn);
  if (p->window > 0) steps = std::min(steps, cdiv(p->window + most, own.s.bn) + 1);
  // two blocks of the kernel over keys run on a CU: 512 pieces would be one round, but twice as many even out
  // unequal lengths (40 sequences of 1 to 4096 tokens: 41.7 us against 46.9)
  const int64_t target = own.s.pair ? 768 : 1024, tiles = slots * Hkv;
  const int64_t room = own.s.keys ? cdiv(2 * target, tiles) : target / tiles;
  int64_t splits = std::max<int64_t>(1, std::min<int64_t>({room, steps, 64}));

  // the prefix: its length is known here, so its pieces are too
  int64_t sp = 0;
  if (shared) {
    pre.a = a;
    choose_shape(pre.s, n * G, n * G * Hkv, p->dt, D, BS, a.sb_bytes != 0, gqa_cap_needs_tanh(a));
    pre.a.shared = 1;
    pre.a.front = (int)std::min<int64_t>(p->prefix_len, p->prefix_count * BS);
    pre.a.bt = p->prefix_blocks, pre.a.bt_ss = 0;
    pre.a.bm_log = __builtin_ctz(pre.s.bm);
    pre.a.bn_log = __builtin_ctz(pre.s.bn);
    pre.a.slots = (int)cdiv(n * G, 1ll << pre.a.bm_log);
    const int64_t pt = pre.a.slots * Hkv, ps = std::max<int64_t>(cdiv(pre.a.front, pre.s.bn), 1);
    // a block a CU, or two: half of it leaves CUs idle (64 sequences behind 8192 tokens, 256 rows a K/V head: 67 us
    // against 58), the smaller tiles' kernel with two blocks a CU takes as long (57) and 256 of them longer (63)
    const int64_t ptarget = pre.s.pair ? 256 : 512;
    sp = std::max<int64_t>(1, std::min<int64_t>({ptarget / pt, ps, 48}));
    pre.a.splits = (int)sp;
    splits = std::min<int64_t>(splits, 64 - sp);
    pre.blocks = pt * sp;
  }
  const int64_t pieces = sp + splits, rows = T * Hkv * G;
  own.a.slots = (int)slots;
  own.a.splits = (int)splits;
  own.a.piece0 = (int)sp;
  own.a.pieces = (int)pieces;
  own.a.cap_tiles = (int)std::max<int64_t>(cdiv(2048, own.s.bn), cdiv(steps, splits));
  own.a.target = (float)target;
  own.blocks = slots * Hkv * splits;
  pre.a.pieces = (int)pieces;
  if (slots > 0x3FFFFFFF || own.blocks > 0x7FFFFFFF || pre.blocks > 0x7FFFFFFF) return fail(MLS_ERR_UNSUPPORTED, "%s: too large", fn);
  need = pieces > 1 ? rows * (pieces * (a.DW + 2) + 1) : 0;
  if (need == 0) ws = nullptr;  // (one piece writes no records and no counts, also where a workspace is given)
  own.a.ws = pre.a.ws = ws;
  own.a.ws_ml = pre.a.ws_ml = ws ? ws + rows * pieces * a.DW : nullptr;
  own.a.ws_live = ws ? reinterpret_cast<int32_t*>(ws + rows * pieces * (a.DW + 2)) : nullptr;
  return MLS_OK;
}

int launch(int dt, const Pass& p, hipStream_t st) {
  if (dt == MLS_F32) return gqa_launch<float>(p.a, p.s, p.blocks, st);
  if (dt == MLS_F16) return gqa_launch<_Float16>(p.a, p.s, p.blocks, st);
  return gqa_launch<__bf16>(p.a, p.s, p.blocks, st);
}

}  // namespace

}  // namespace mls

using namespace mls;

extern "C" int64_t mlsx_paged_attention_ws(const mlsx_paged_attention_args* p) {
  Pass own, pre;
  bool shared;
  int64_t need;
  if (!p || prepare("mlsx_paged_attention", p, nullptr, own, pre, shared, need) != MLS_OK) return 0;
  return need;
}

extern "C" int mlsx_paged_attention(const mlsx_paged_attention_args* p, float* workspace, int64_t workspace_floats,
                                    mls_stream_t stream) {
  const char* fn = "mlsx_paged_attention";
  if (!p) return fail(MLS_ERR_ARG, "%s: null arguments", fn);
  Pass own, pre;
  bool shared;
  int64_t need;
  int rc = prepare(fn, p, workspace, own, pre, shared, need);
  if (rc != MLS_OK || own.blocks == 0) return rc;
  if (need > 0 && (!workspace || workspace_floats < need))
    return fail(MLS_ERR_ARG, "%s: workspace of %lld floats needed (mlsx_paged_attention_ws)", fn, (long long)need);
  if (need > 0 && !aligned(workspace, 16)) return fail(MLS_ERR_ARG, "%s: workspace not 16-byte aligned", fn);
  hipStream_t st = (hipStream_t)stream;
  if (shared && (rc = launch(p->dt, pre, st)) != MLS_OK) return rc;
  if ((rc = launch(p->dt, own, st)) != MLS_OK) return rc;
  if (own.a.pieces == 1) return MLS_OK;
  if (p->dt == MLS_F32) return launch_join<float>(own.a, st);
  if (p->dt == MLS_F16) return launch_join<_Float16>(own.a, st);
  return launch_join<__bf16>(own.a, st);
}
