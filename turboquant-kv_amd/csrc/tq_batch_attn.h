// tq_batch_attn.h -- attention of a ragged batch over decode-layout paged pools on gfx950:
// the kernel (instantiated per value width by tq_batch_attn_v{2,3,4}.hip) and its schedule.
//
// Semantics.  Sequence b's new tokens are rows query_start[b] .. query_start[b + 1] - 1 of q,
// at positions p = T_b - n_b + i of its T_b = seq_lens[b] tokens.  A token sees the positions
//   max(token_start, p - window + 1) <= j < min(T_b, max(p + 1, prefix_len_b))
// (a part that is not given does not bound).  score = scale <q, k_j>, then softcap *
// tanh(score / softcap), then + slope_h (j - p); softmax over the visible positions, and
// out = sum_j w_j v_j.  k_j = n_j c[code] R_k, so scores are taken against R_k q; the weighted
// sum is rotated back by R_v once.  A row that sees nothing gives zeros and lse = -inf.
//
// Split kernel (few rows).  The work is a line of 64-token tiles: for each item (16 NGR query
// rows of one sequence: row r is query head h G + r % G of new token r / G) its tiles, once per
// KV head.  Workgroup w takes the w-th of equal pieces of that line, whatever the lengths: its
// eight waves take a piece's tiles in turn and merge in LDS; an item cut between workgroups
// leaves partial sums in its workgroups' slots, which the combine kernel joins.  Every
// workgroup finds its place in the line itself from the device lengths.
// Row kernel (prompts).  A wave per 16 NGR rows streams all tiles they see.
//
// Per tile, wave and group of 16 rows (the scheme of the prefill kernel):
//   S^T = K Qrot^T  v_mfma_f32_16x16x32_f16 per 16-token group b and half s of the dims.  A: lane
//                   (c, g) = (lane % 16, lane / 16) holds token 16 b + c, dims 16 g + 8 s .. + 7:
//                   four bytes of its key row, each one table lookup of (c[hi], c[lo]).  B: the
//                   rotated query.  Lane (c, g) gets tokens 16 b + 4 g + r of query row c.
//   O^T += V^T P^T  A: value centroids of dim 16 nb + c for the tokens the lane holds weights of,
//                   looked up by the bytes of its value words.  B: weights times value norms.
// Tables: 256 entries of 256 B for keys and for values (copies of each entry over all 64 banks,
// so that lookups do not collide), one v_perm_b32 per address: 128 KB, built once per workgroup.
// Tiles are loaded two ahead; a tile's norms (one per lane) reach the lanes through LDS.
// fp32 / fp16 queries: fp16 hi + lo parts of every operand (three products per term, about
// 2^-22 relative); bf16 queries: one product per term (2^-11 relative per operand, below the
// bf16 rounding of their outputs).  Sums, statistics and rotations are fp32.
#pragma once

#include "tq_common.h"

#include <climits>
#include <type_traits>

namespace tq {

constexpr int kBaWaves = 8;
constexpr int kBaThreads = 64 * kBaWaves;
// Row groups of a wave where rows abound: with hi + lo parts two fit the registers.
constexpr int ba_groups(bool prec) { return prec ? 2 : 3; }
// Floats of a partial slot of R rows: sums [R][64], (maximum, sum) [R][2].
constexpr int ba_slot_floats(int R) { return R * 66; }

// What the schedule leaves for the combine kernel.
struct BaHead {
  int64_t chunk;  // tiles per workgroup
  int32_t n_items;
  int32_t pad;
};
struct BaItem {
  int64_t start;  // place of its first tile on the line (KV head h: + h * cost)
  int32_t cost;
  int32_t seg, rt;
  int32_t pad;
};

struct BaArgs {
  const void* q;
  int64_t q_stride;  // elements between tokens
  int q_dt;
  int n_tokens, hq, hkv, G, B;
  const int32_t* query_start;  // [B + 1]
  const int32_t* seq_lens;     // [B]
  const int32_t* group_start;  // [n_groups + 1], or null
  const int32_t* shared;       // [n_groups]
  int n_groups;
  int over_groups;             // this launch's segments: the groups' shared tokens
  const uint8_t* kpairs;       // [num_blocks][hkv][bs][32]
  const float* knorms;         // [num_blocks][hkv][bs]
  const uint8_t* vtiles;       // [num_blocks][hkv][bs/64][512 VB] or [num_blocks][hkv][bs/16][128 VB]
  const float* vnorms;
  const int32_t* block_tables;
  int64_t table_stride;
  int max_blocks, bs_log2;
  uint32_t num_blocks;
  int cap;                     // tokens a table row holds, at most INT_MAX - 127
  const float* kcen;
  const float* vcen;
  const float* krot;
  const float* vrot;
  float qscale;                // softmax scale * log2(e)
  float cap2, cap2_inv;        // softcap * log2(e) and its inverse, or 0
  const float* slopes;         // [hq] or null
  int window;                  // 0: none
  const int32_t* prefix_lens;  // [B] or null
  const int32_t* token_starts; // [n_tokens] or null
  void* out;
  int64_t out_stride;
  float* lse;                  // [n_tokens][hq] or null
  int zero_tail;               // rows behind the last sequence get zeros
  // partial results: of the pieces of cut items, and (with groups) of whole ones by row
  float* slots;                // [grid][2][ba_slot_floats(R)]
  BaHead* head;
  BaItem* items;
  int max_items;               // entries of `items`
  int32_t* seg_item;           // [n_groups]: first item of each group
  float* row_sums;             // [n_tokens * hq][64], or null: whole items are written to out
  float* row_stats;            // [n_tokens * hq][2]
};

typedef float ba_v4f __attribute__((ext_vector_type(4)));
typedef _Float16 ba_v8h __attribute__((ext_vector_type(8)));
typedef uint32_t ba_u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t ba_u32x2 __attribute__((ext_vector_type(2)));

// Launches the kernel of value width VB; rows: the row kernel (grid workgroups of one item and
// KV head each), else the split kernel with ba_groups(prec) or one group of rows a wave.
template <int VB>
void ba_launch(const BaArgs& a, bool sub, bool prec, bool rows, int groups, unsigned grid, hipStream_t st);
extern template void ba_launch<2>(const BaArgs&, bool, bool, bool, int, unsigned, hipStream_t);
extern template void ba_launch<3>(const BaArgs&, bool, bool, bool, int, unsigned, hipStream_t);
extern template void ba_launch<4>(const BaArgs&, bool, bool, bool, int, unsigned, hipStream_t);

// ------------------------------------------------------------------------------- schedule

// A segment: the rows of a sequence (or, over groups, of a group's sequences) and the
// positions they are taken over here.
struct BaSeg {
  int tok0, ntok;  // tokens of q
  int past;        // position of the first (sequences)
  int lo, hi;      // positions this launch covers
  int prefix;      // prefix_lens
  int table;       // row of block_tables
  int b0, b1;      // sequences (groups)
  int nrt;         // items
};

__device__ __forceinline__ int ba_qs(const BaArgs& a, int b) {
  return max(0, min(a.query_start[b], a.n_tokens));
}

// The last i < n with key(i) <= v, keys ascending; 0 if there is none.
template <typename F>
__device__ __forceinline__ int ba_last(int n, int v, F key) {
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (key(mid) <= v) lo = mid;
    else hi = mid;
  }
  return lo;
}

// Tokens of sequence b's context that its group's launch covers.
__device__ __forceinline__ int ba_shared(const BaArgs& a, int b) {
  if (!a.group_start || a.n_groups == 0) return 0;
  const int g = ba_last(a.n_groups, b, [&](int i) { return a.group_start[i]; });
  if (b < a.group_start[g] || b >= a.group_start[g + 1]) return 0;
  return max(0, min(a.shared[g], a.cap));
}

__device__ __forceinline__ BaSeg ba_segment(const BaArgs& a, int s, int rows) {
  BaSeg x{};
  if (a.over_groups) {
    x.b0 = max(0, min(a.group_start[s], a.B));
    x.b1 = max(x.b0, min(a.group_start[s + 1], a.B));
    x.hi = max(0, min(a.shared[s], a.cap));
    if (x.b1 > x.b0 && x.hi > 0) {
      x.tok0 = ba_qs(a, x.b0);
      x.ntok = max(0, ba_qs(a, x.b1) - x.tok0);
    }
    x.table = min(x.b0, a.B - 1);
  } else if (s < a.B) {
    x.tok0 = ba_qs(a, s);
    x.ntok = max(0, ba_qs(a, s + 1) - x.tok0);
    const int T = max(0, a.seq_lens[s]);
    x.past = T - x.ntok;
    x.lo = ba_shared(a, s);
    x.hi = min(T, a.cap);
    x.prefix = a.prefix_lens ? a.prefix_lens[s] : 0;
    x.table = s;
  } else {  // rows behind the last sequence: they see nothing
    x.tok0 = a.B ? ba_qs(a, a.B) : 0;
    x.ntok = a.n_tokens - x.tok0;
  }
  x.nrt = (int)(((int64_t)x.ntok * a.G + rows - 1) / rows);
  return x;
}

// First tile and number of tiles of item rt.  Document starts bound it for single tokens; the
// waves of longer items skip the tiles that their own rows' starts leave out.
__device__ __forceinline__ void ba_range(const BaArgs& a, const BaSeg& x, int rt, int rows, int& t0, int& nt) {
  int64_t lo = x.lo, hi = x.hi;
  if (!a.over_groups) {
    const int i0 = (int)((int64_t)rt * rows / a.G);
    const int i1 = min(x.ntok - 1, (int)(((int64_t)rt * rows + rows - 1) / a.G));
    hi = min<int64_t>(hi, max<int64_t>((int64_t)x.past + i1 + 1, x.prefix));
    if (a.window > 0) lo = max<int64_t>(lo, (int64_t)x.past + i0 + 1 - a.window);
    if (a.token_starts && x.ntok == 1 && hi > 0) lo = max<int64_t>(lo, a.token_starts[x.tok0]);
  }
  t0 = hi > lo ? (int)(lo >> 6) : 0;
  nt = hi > lo ? (int)((hi + 63) >> 6) - t0 : 0;
}

// A place on the line: item rt of segment seg, `at` tiles into its hkv * cost.
struct BaPlace {
  int seg, rt, item;
  int64_t at;
};

}  // namespace tq
