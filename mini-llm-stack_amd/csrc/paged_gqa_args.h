// Arguments of the paged grouped-head attention kernels, and which rows, keys and pieces of a
// context a block takes (found on the device: the host knows neither lengths nor offsets).
#pragma once

#include "common.h"

namespace mls {

struct GqaArgs {
  const void* q;  // [T][Hkv * group][D], strides (q_st, q_sh, 1)
  int64_t q_st, q_sh;
  const void* kp;  // [num_blocks][Hkv][BS][D], strides (kv_sb, kv_sh, kv_st, 1), as vp
  const void* vp;
  int64_t kv_sb, kv_sh, kv_st;
  const int32_t* bt;  // [n][max_blocks]; shared: [max_blocks]
  int64_t bt_ss;
  const int32_t* lens;    // [n] keys of each sequence, its new tokens among them
  const int32_t* cu;      // [n + 1] first row of each sequence; null: one row each
  const int32_t* prefix;  // [n] or null: keys that every row sees, also before it
  const float* slopes;    // [Hkv * group] or null
  void* out;
  int64_t o_st, o_sh;
  float* ws;     // [T][Hkv * group][pieces][DW]: O of each piece, not divided by its sum
  float* ws_ml;  // [T][Hkv * group][pieces][2]: its reference and sum
  int32_t* ws_live;  // [T][Hkv * group]: pieces of the sequence's own keys that were made
  int64_t num_blocks;
  int n, T, Hkv, group, D, DW, BS;
  uint32_t bs_magic;  // ceil(2^32 / BS)
  uint32_t sb_bytes, st_bytes;  // kv_sb, kv_st in bytes where they fit (0: not)
  int max_keys;           // a table's tokens
  int window;
  int front;   // shared: keys of the prefix
  int shared;  // the rows of all sequences (one each) over the one table's `front` keys
  float c, cap, to_cap;  // scale log2(e); cap log2(e) (0: none), scale / cap
  int simple;            // scores are positive multiples of the products: no cap, no slopes
  int bm_log, bn_log;    // rows of a tile and keys of a step (log2)
  int slots;             // row tiles that the grid has room for
  int pieces;            // records a row has in the workspace
  int piece0;            // first record of this launch's pieces (before it: the shared prefix's)
  int splits, cap_tiles;  // pieces a context may have; n > 1024: steps of one
  float target;                  // blocks to aim at
  int q_vec, o_vec, kv_vec;  // 16-byte accesses of q, 4 elements at once of out, 16-byte ones of the pools
};

// 16-bit types: 1 - 2 / (e^2y + 1) is off by up to 2^-22, so a score by 2^-22 of the cap, for small scores too: at a cap of
// 256 an eighth of what rounding a weight to fp16 leaves. Past that the scores take tanhf, precise relative to y, and the
// paired kernel, which it would slow with any cap (chunks of D = 256, cap 30: 145 us against 138), is not taken (prompt of
// 8192, cap 300: 1379 us against 1277 there; cap 50: 879).
__host__ __device__ __forceinline__ bool gqa_cap_needs_tanh(const GqaArgs& a) { return a.cap > 256.0f * 1.44269504f; }

struct GqaShape {
  bool keys, pair, vec;
  int nt, dp, bn, bm;
  int group_rows;  // cache rows that one load instruction covers: of one block each, where vec
};

struct GqaPlan {
  const int32_t* table;
  int tok0, rows, row0;  // the sequence's first row of q, its packed rows, the tile's first of them
  int pos0, len, pfx;    // position of its first new token; its keys; keys seen both ways
  int klo, khi;          // keys that any row of the tile sees
  int lo, tiles;         // the tile's first step, steps
  int live, per;         // pieces, steps of a piece
  bool direct;           // the only piece writes the output itself
};

// key / BS
__device__ __forceinline__ int gqa_block_of(const GqaArgs& a, int key) {
  const uint32_t b = a.BS == 1 ? (uint32_t)key : __umulhi((uint32_t)key, a.bs_magic);  // (one too many at most)
  return (int)(b - (b * (uint32_t)a.BS > (uint32_t)key ? 1 : 0));
}

// The last s of [0, n] whose start(s) is at most `at`, -1: none; by 64 probes a round.
template <typename F>
__device__ __forceinline__ int last_start(int n, int at, int lane, F start) {
  int lo = 0, hi = n + 1;
  while (true) {
    const int step = (hi - lo + 63) / 64, s = lo + lane * step;
    const bool le = s < hi && start(s) <= at;
    const int cnt = __builtin_popcountll(__ballot(le));
    if (cnt == 0) return lo - 1;  // (only in the first round, where starts rise)
    lo += (cnt - 1) * step;
    if (step == 1) return lo;
    hi = min(lo + step, hi);
  }
}

__device__ __forceinline__ int gqa_cu(const GqaArgs& a, int s) { return min(max(a.cu[s], 0), a.T); }

// First slot of sequence s's row tiles (s = n: the rows past the last sequence's): room for any
// lengths without a prefix sum, since floor(x) + 1 >= ceil(x).
__device__ __forceinline__ int gqa_slot_of(const GqaArgs& a, int s) {
  return (int)(((int64_t)gqa_cu(a, s) * a.group) >> a.bm_log) + s + 1;
}

// The sequence of a slot, or of a row of q.
template <bool SLOT>
__device__ __forceinline__ int gqa_find(const GqaArgs& a, int at, int lane) {
  return last_start(a.n, at, lane, [&](int s) { return SLOT ? gqa_slot_of(a, s) : gqa_cu(a, s); });
}

__device__ __forceinline__ int gqa_keys_of(const GqaArgs& a, int s) {
  return min(max(a.lens[s], 0), a.max_keys);
}

// Steps of a piece: what makes about `target` blocks of the batch's own lengths, and at most
// `splits` pieces of the longest. Every wavefront of both kernels finds the same. Past 1024 sequences (one K/V head, or the host
// leaves no room for pieces) the sum takes longer than even pieces save: 1100 of 1 to 4096 tokens, 8 heads, 104 us with
// steps of a fixed number, 109 with the sum; 2000 of them 157 / 177, of 10 to 300 tokens 36.5 / 47.4.
__device__ __forceinline__ int gqa_piece(const GqaArgs& a, int lane) {
  if (a.n > 1024) return a.cap_tiles;
  float sum = 0.0f;
  int most = 0;
  for (int s = lane; s < a.n; s += 64) {
    const int nt = a.cu ? max(gqa_cu(a, s + 1) - gqa_cu(a, s), 0) : 1;
    uint32_t keys = gqa_keys_of(a, s);
    if (a.window > 0) keys = min(keys, (uint32_t)a.window + nt);
    const int t = (int)((keys + (1u << a.bn_log) - 1) >> a.bn_log);
    sum += (float)((nt * a.group + (1 << a.bm_log) - 1) >> a.bm_log) * (float)t;
    if (nt > 0) most = max(most, t);
  }
  sum = lane_group_sum<64>(sum);
  most = (int)lane_group_max<64>((float)min(most, 1 << 24));
  const int want = (int)fminf(ceilf(sum * a.Hkv / a.target), 1e9f);
  return __builtin_amdgcn_readfirstlane(max(max(want, (most + a.splits - 1) / a.splits), 1));
}

// First key within the window of a row at `pos` (which may be far below 0, and the window up to 2^31 - 1)
__device__ __forceinline__ int gqa_window_from(const GqaArgs& a, int pos) {
  return a.window > 0 && pos >= a.window ? pos - a.window + 1 : 0;
}

// Shared: the position of sequence s's row, behind the prefix; at most 2^31 - 2, for any length
__device__ __forceinline__ int gqa_shared_pos(const GqaArgs& a, int s) {
  return (int)min((uint32_t)a.front + (uint32_t)max(a.lens[s], 0), 0x7FFFFFFFu) - 1;
}

// Row tile rt of sequence seq (-1 and n: rows that no sequence holds, which see nothing), for its piece `split`.
__device__ __forceinline__ GqaPlan gqa_tile_plan(const GqaArgs& a, int seq, int rt, int split, int lane) {
  GqaPlan p;
  const bool real = seq >= 0 && seq < a.n;
  int ntok;
  if (a.shared) {
    p.tok0 = 0;
    ntok = a.n;
    p.pos0 = 0;
    p.len = a.front;
  } else {
    p.tok0 = a.cu ? (seq < 0 ? 0 : gqa_cu(a, seq)) : seq;
    ntok = a.cu ? max((seq >= a.n ? a.T : gqa_cu(a, seq + 1)) - p.tok0, 0) : 1;
    p.pos0 = real ? a.lens[seq] - ntok : 0;
    p.len = real ? gqa_keys_of(a, seq) : 0;
  }
  p.pfx = real && a.prefix ? a.prefix[seq] : 0;
  p.table = a.bt + (a.shared || !real ? 0 : seq * a.bt_ss);
  p.rows = ntok * a.group;
  p.live = p.tiles = p.per = 0;
  p.klo = p.khi = p.lo = 0;
  p.direct = false;
  // (offsets that do not rise can lead the search to a sequence that begins behind the slot: rt < 0)
  if ((uint32_t)rt >= (uint32_t)(p.rows + (1 << a.bm_log) - 1) >> a.bm_log) {
    p.row0 = p.rows = 0;
    return p;
  }
  p.row0 = rt << a.bm_log;
  const int first = p.row0 / a.group, last = (min(p.row0 + (1 << a.bm_log), p.rows) - 1) / a.group;
  int pmin, pmax;
  if (a.shared) {
    pmin = 0x7FFFFFFF;
    pmax = a.front - 1;
    if (a.window > 0) {
      for (int t = first + lane; t <= last; t += 64) pmin = min(pmin, gqa_shared_pos(a, t));
#pragma unroll
      for (int off = 32; off >= 1; off >>= 1) pmin = min(pmin, __shfl_xor(pmin, off, 64));
    }
  } else {
    pmin = p.pos0 + first;
    pmax = p.pos0 + last;
  }
  p.khi = __builtin_amdgcn_readfirstlane(min(max(pmax + 1, p.pfx), p.len));
  p.klo = __builtin_amdgcn_readfirstlane(gqa_window_from(a, pmin));
  p.lo = p.klo >> a.bn_log << a.bn_log;
  p.tiles = p.khi > p.klo ? (int)(((uint32_t)(p.khi - p.lo) + (1u << a.bn_log) - 1) >> a.bn_log) : 0;
  if (a.shared) {
    p.live = a.splits;
  } else if (a.splits > 1 && p.tiles > max(split, 1)) {  // (a piece has a step or more: others need no lengths of the batch)
    const int piece = gqa_piece(a, lane);
    p.live = min(max((p.tiles + piece - 1) / piece, 1), a.splits);
  } else {
    p.live = 1;
  }
  p.per = (p.tiles + p.live - 1) / p.live;
  p.direct = p.live == 1 && a.pieces == 1;
  if (!a.shared && a.piece0 == 0 && p.live == 1) p.direct = true;
  return p;
}

// Block -> (K/V head, piece, row tile). Heads run fastest: with 8 of them, blocks go round the 8
// XCDs in order, so that an XCD's L2 holds one head's keys. The later row tiles, which see more
// keys, come first; the pieces that few sequences reach last.
__device__ __forceinline__ GqaPlan gqa_block_plan(const GqaArgs& a, int block, int lane, int& kvh, int& split) {
  kvh = block % a.Hkv;
  const int rest = block / a.Hkv;
  split = rest / a.slots;
  const int slot = a.slots - 1 - rest % a.slots;
  if (a.shared) return gqa_tile_plan(a, 0, slot, split, lane);
  if (!a.cu) {
    const int per = (a.group + (1 << a.bm_log) - 1) >> a.bm_log;
    return gqa_tile_plan(a, slot / per, slot % per, split, lane);
  }
  const int seq = __builtin_amdgcn_readfirstlane(gqa_find<true>(a, slot, lane));
  return gqa_tile_plan(a, seq, seq < 0 ? slot : slot - __builtin_amdgcn_readfirstlane(gqa_slot_of(a, seq)), split, lane);
}

// The keys [lo, hi) that the row of token `tok` sees, and its position.
__device__ __forceinline__ void gqa_row_range(const GqaArgs& a, const GqaPlan& p, int tok, int& lo, int& hi, int& pos) {
  pos = a.shared ? gqa_shared_pos(a, tok) : p.pos0 + (tok - p.tok0);
  hi = min(max(pos + 1, p.pfx), p.len);
  lo = gqa_window_from(a, pos);
}

// Over the packed rows r0 .. r1 (none where r1 < r0) of one sequence, or of shared rows: the extremes
// of the keys [lo, hi) that they see.
__device__ __forceinline__ void gqa_wave_range(const GqaArgs& a, const GqaPlan& p, int r0, int r1, int lane, int& lo_min,
                                               int& lo_max, int& hi_min, int& hi_max) {
  lo_min = hi_min = 0x7FFFFFFF;
  lo_max = hi_max = -0x7FFFFFFF;
  if (r1 < r0) return;
  const int t0 = p.tok0 + r0 / a.group, t1 = p.tok0 + r1 / a.group;
  if (!a.shared) {  // (positions rise with the row)
    int pos;
    gqa_row_range(a, p, t0, lo_min, hi_min, pos);
    gqa_row_range(a, p, t1, lo_max, hi_max, pos);
    return;
  }
  hi_min = hi_max = p.len;
  lo_min = lo_max = 0;
  if (a.window <= 0) return;
  int lo, hi, pos;
  gqa_row_range(a, p, min(t0 + lane, t1), lo, hi, pos);  // (at most 32 rows)
  lo_min = lo_max = lo;
#pragma unroll
  for (int off = 32; off >= 1; off >>= 1) {
    lo_min = min(lo_min, __shfl_xor(lo_min, off, 64));
    lo_max = max(lo_max, __shfl_xor(lo_max, off, 64));
  }
  lo_min = __builtin_amdgcn_readfirstlane(lo_min);
  lo_max = __builtin_amdgcn_readfirstlane(lo_max);
}

}  // namespace mls
