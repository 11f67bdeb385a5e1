// tq_batch_attn.h -- attention of a ragged batch over decode-layout paged pools on gfx950:
// the kernel (tq_batch_attn_kernel.h, instantiated per value width and pool by
// tq_batch_attn_{2,3,4}{t,s}.hip) and its schedule.
//
// Semantics.  Sequence b's new tokens are rows query_start[b] .. query_start[b + 1] - 1 of q,
// at positions p = T_b - n_b + i of its T_b = seq_lens[b] tokens.  A token sees the positions
//   max(token_start, p - window + 1) <= j < min(T_b, max(p + 1, prefix_len_b))
// (a part that is not given does not bound).  score = scale <q, k_j>, then softcap *
// tanh(score / softcap), then + slope_h (j - p); softmax over the visible positions, and
// out = sum_j w_j v_j.  k_j = n_j c[code] R_k, so scores are taken against R_k q; the weighted
// sum is rotated back by R_v once.  A row that sees nothing gives zeros and lse = -inf.
//
// Schedule.  The work is a line of 64-token tiles: for each item (R query rows of one sequence:
// row r is query head h G + r % G of new token r / G) its tiles, once per KV head, each (item,
// head) preceded by kBaOver places that stand for what it costs besides its tiles.  Wave w of
// the grid takes the w-th of equal pieces of that line, whatever the lengths are: no wave waits
// for another.  A wave that takes all of an (item, head) leaves its sums by row, one that takes
// a part leaves them in a slot of its own; the joining kernel adds them up and rotates the result.
// Items of many rows are mostly one wave's: without groups that wave rotates and writes their
// results itself, and only cut items are joined.
// With groups, the shared prefixes are a second line whose items hold the rows of all the
// group's sequences: each of their tiles is read once for R rows of the group.
// A preparing kernel rotates the queries, finds every token's positions and lays the line out
// from the device lengths, so the waves of the main kernel start from two dependent loads.
//
// Per tile, wave and group of 16 columns (NGR groups share a tile's lookups):
//   S^T = K Qrot^T  v_mfma_f32_16x16x32_f16 per 16-token group b and half s of the dims.  A: lane
//                   (c, g) = (lane % 16, lane / 16) holds token 16 b + c, dims 16 g + 8 s .. + 7:
//                   four bytes of its key row, each one table lookup of (c[hi], c[lo]).  B: the
//                   rotated query of column c.  Lane (c, g) gets tokens 16 b + 4 g + r.
//   O^T += V^T P^T  A: value centroids of dim 16 nb + c for the tokens the lane holds weights of,
//                   looked up by the bytes of its value words.  B: weights times value norms.
// Few rows (RW = 4 or 8 of the 16 columns: single tokens): the columns are 16 / RW copies of the
// rows, and copy k keeps only the scores of its own share of a tile's tokens (a select after
// the first products), so a lane's softmax handles RW / 4 * 4 scores instead of 16; the weights
// of the other copies' tokens are zeros in the second products, and the copies' maxima, sums and
// outputs are joined when the wave is done.
// Tables: 256 entries of 256 B for keys and for values (copies of each entry over all 64 banks,
// so that lookups do not collide), one v_perm_b32 per address: 128 KB, built once per workgroup.
// Tiles are loaded ahead in registers; a tile's norms (one per lane) reach the lanes through LDS.
// fp32 / fp16 queries: fp16 hi + lo parts of every operand (three products per term, about
// 2^-22 relative); bf16 queries: one product per term (2^-11 relative per operand, below the
// bf16 rounding of their outputs).  Sums, statistics and rotations are fp32.
#pragma once

#include "tq_common.h"

#include <climits>
#include <type_traits>

namespace tq {

// Waves of a workgroup (one per CU: the tables fill its LDS).  256 registers a wave; 12 waves of 168
// were no faster (48 sequences of up to 32k tokens: 89 and 91 us) and leave more to be joined.
constexpr int kBaWaves = 8;
constexpr int kBaMaxSegs = 8192;  // sequences or groups of a call: the preparing kernel's LDS
constexpr int kBaQueryTop = 14;   // rotated queries are scaled to at most 2^14 (fp16's range ends at 2^16)
constexpr int kBaOver = 3;        // an (item, head)'s cost besides its tiles, in tiles
// Groups of 16 rows that a wave takes where rows abound.  Three share a tile's lookups best where
// their registers allow (bf16 queries without prefix groups: prompts 446 -> 395 us for three
// spilling 40 values outside the loop; beside a second line 60 -> 63 us).
constexpr int ba_groups(bool prec, bool pair) { return prec || pair ? 2 : 3; }
// Floats of a partial slot of R rows: sums [R][64], (maximum, sum) [R][2].
constexpr int ba_slot_floats(int R) { return R * 66; }

// A line of work as the preparing kernel lays it out.
struct BaHead {
  int64_t chunk, total;  // places of a wave's piece, of the line
  int32_t n_items, pieces;
};
struct BaItem {
  int64_t start;      // its first place (KV head h: + h * (nt + kBaOver))
  int32_t t0, nt;     // tiles
  int32_t tok0;       // its segment's first token, its first row and the segment's rows
  int32_t row0, nrows;
  int32_t table;      // row of block_tables
  int32_t lo, hi;     // positions this line covers
};
// An entry of the tables: byte i's key centroids (c[i / 16], c[i % 16]) and value centroids as
// fp16 hi and lo parts, scaled by powers of two into [0.5, 1).
struct BaEntry {
  uint32_t khi, klo, vhi[2], vlo[2];
  float vsc_inv;  // the values' scale undone
  uint32_t pad;
};
struct BaLine {
  BaHead* head;
  BaItem* items;
  int32_t max_items;   // entries of `items`
  int32_t* seg_item;   // [segments + 1]: first item of each
  int32_t* work;       // [waves]: the item that the wave's piece begins in; -1: behind the line's end
  int32_t waves;
  int32_t rows;        // R
  float* slots;        // [waves][2][ba_slot_floats(R)]
  float* row_sums;     // [n_tokens * hq][64] (not where waves write results)
  float* row_stats;    // [n_tokens * hq][2]
};
// A token's visible positions, its own, and its sequence (B: behind the last).
struct BaToken {
  int32_t lo, hi, pos, seq;
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
  int krot_row, krot_col, vrot_row, vrot_col;  // strides of their rows and columns
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
  // made by the preparing kernel
  _Float16* qhi;               // [n_tokens * hq][64] rotated queries over a power of two: hi,
  _Float16* qlo;               // and lo parts (fp32 / fp16 queries)
  int32_t* qexp;               // [n_tokens * hq] log2 of what undoes it and the key centroids' scale
  BaEntry* entries;            // [256]
  _Float16* vrot16;            // R_v's operands, [2 parts][4 ob][2 s][64 lanes][8]: see ba_rotate_back
  int direct;                  // (no groups) waves write the results of whole items of many rows
  BaToken* tokens;             // [n_tokens]
  BaLine line[2];              // sequences, groups
};

typedef float ba_v4f __attribute__((ext_vector_type(4)));
typedef _Float16 ba_v8h __attribute__((ext_vector_type(8)));
typedef uint32_t ba_u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t ba_u32x2 __attribute__((ext_vector_type(2)));

// Launches the main kernel of value width VB over line 0, or (pair) both lines (rw: 4, 8 or 16 rows
// a group of columns; SUB: pools of 16-token value sub-blocks; wide: pools of 4 GB and more).
template <int VB, bool SUB>
void ba_launch(const BaArgs& a, bool pair, bool wide, bool prec, int rw, int groups, unsigned grid, hipStream_t st);
#define BA_LAUNCH(VB, SUB) \
  template void ba_launch<VB, SUB>(const BaArgs&, bool, bool, bool, int, int, unsigned, hipStream_t);
extern BA_LAUNCH(2, false) extern BA_LAUNCH(2, true)
extern BA_LAUNCH(3, false) extern BA_LAUNCH(3, true)
extern BA_LAUNCH(4, false) extern BA_LAUNCH(4, true)

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

// a / b for 0 <= a, 0 < b: places rarely need 64 bits, whose division takes ten times as long.
__device__ __forceinline__ int64_t ba_div(int64_t a, int64_t b) {
  return ((a | b) >> 32) == 0 ? (int64_t)((uint32_t)a / (uint32_t)b) : a / b;
}

// The rows' results from their sums: out_c[16 ob + 4 g + r] of lane (c, g), c the row, in fp16
// products over 32 dims: part s's operands are A[c][8 g + i] = R_v[dim][16 ob + c] and B[8 g + i][c]
// = x_c[dim] with dim = 16 (2 s + i / 4) + 4 g + i % 4, the dims that lane (c, g) holds in
// x[2 s + i / 4][i % 4].  PREC: hi + lo parts of both.  |x| at most 2^15.
template <bool PREC>
__device__ __forceinline__ void ba_rotate_back(const _Float16* vrot16, const ba_v4f* x, int lane, ba_v4f* out) {
  ba_v8h hi[2], lo[2];
#pragma unroll
  for (int s = 0; s < 2; ++s)
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if constexpr (PREC) {
        _Float16 hv, lv;
        split_f16(x[2 * s + (i >> 2)][i & 3], hv, lv);
        hi[s][i] = hv;
        lo[s][i] = lv;
      } else {
        hi[s][i] = (_Float16)x[2 * s + (i >> 2)][i & 3];
      }
    }
  if constexpr (PREC) mfma_operand_fence(hi[0], hi[1], lo[0], lo[1]);
  else mfma_operand_fence(hi[0], hi[1]);
#pragma unroll
  for (int ob = 0; ob < 4; ++ob) {
    out[ob] = (ba_v4f){0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      const ba_v8h* src = reinterpret_cast<const ba_v8h*>(vrot16) + (ob * 2 + s) * 64 + lane;
      const ba_v8h ah = src[0];
      out[ob] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ah, hi[s], out[ob], 0, 0, 0);
      if constexpr (PREC) {
        const ba_v8h al = src[512];
        out[ob] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ah, lo[s], out[ob], 0, 0, 0);
        out[ob] = __builtin_amdgcn_mfma_f32_16x16x32_f16(al, hi[s], out[ob], 0, 0, 0);
      }
    }
  }
}

// Four dims of a row's result, in the output's type.
__device__ __forceinline__ void ba_store(const BaArgs& a, int tok, int qh, int dim, ba_v4f x) {
  const int64_t at = (int64_t)tok * a.out_stride + qh * 64 + dim;
  if (a.q_dt == TQ_F32) {
    *reinterpret_cast<ba_v4f*>(static_cast<float*>(a.out) + at) = x;
  } else if (a.q_dt == TQ_BF16) {
    typedef __bf16 b4_t __attribute__((ext_vector_type(4)));
    *reinterpret_cast<b4_t*>(static_cast<uint16_t*>(a.out) + at) = __builtin_convertvector(x, b4_t);
  } else {
    typedef _Float16 h4_t __attribute__((ext_vector_type(4)));
    *reinterpret_cast<h4_t*>(static_cast<uint16_t*>(a.out) + at) = __builtin_convertvector(x, h4_t);
  }
}

__device__ __forceinline__ float ba_lse(float m, float l) {
  return l == 0.f ? -INFINITY : (m + __builtin_amdgcn_logf(l)) * 0.6931471805599453f;
}

// Tiles of an (item, head) before place `place` of it.
__device__ __forceinline__ int64_t ba_tiles(int64_t place) { return place > kBaOver ? place - kBaOver : 0; }

}  // namespace tq
