// tq_batch_attn.hip -- entry points of the ragged batch's attention (tq_batch_attn.h): the choice
// of kernels and the workspace, the preparing kernel and the one that joins partial results.

#include "tq_batch_attn.h"

#include <algorithm>

namespace tq {
namespace {

constexpr int kPrepThreads = 512;
constexpr int kPrepWaves = kPrepThreads / 64;
constexpr int kPrepStarts = 2048;  // items' places kept in LDS
constexpr float kBaBalance = 64.f;  // see ba_lay_out's pieces

// ---------------------------------------------------------------------------- preparation

// Exclusive sum over the workgroup; `all` gets the whole sum.
__device__ __forceinline__ int64_t prep_scan(int64_t v, int64_t* part, int64_t* all) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int64_t incl = v;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int64_t up = __shfl_up(incl, o, 64);
    if (lane >= o) incl += up;
  }
  __syncthreads();  // `part` may still be read from a scan before
  if (lane == 63) part[wave] = incl;
  __syncthreads();
  int64_t before = 0, sum = 0;
#pragma unroll
  for (int w = 0; w < kPrepWaves; ++w) {
    const int64_t p = part[w];
    if (w < wave) before += p;
    sum += p;
  }
  *all = sum;
  return before + incl - v;
}

// Tokens of sequence b's context that its group's line covers.
__device__ __forceinline__ int ba_shared(const BaArgs& a, int b) {
  if (a.n_groups == 0) return 0;
  const int g = ba_last(a.n_groups, b, [&](int i) { return a.group_start[i]; });
  if (b < a.group_start[g] || b >= a.group_start[g + 1]) return 0;
  return max(0, min(a.shared[g], a.cap));
}

// A segment of a line: the rows of a sequence or of a group's sequences, the positions the
// line covers, and its table.
struct BaSeg {
  int tok0, ntok, lo, hi, table;
  int past, prefix;  // sequences: the first token's position, prefix_lens
};

template <int L>
__device__ __forceinline__ BaSeg ba_segment(const BaArgs& a, int s) {
  BaSeg x{};
  if (L == 1) {
    const int b0 = max(0, min(a.group_start[s], a.B)), b1 = max(b0, min(a.group_start[s + 1], a.B));
    x.hi = max(0, min(a.shared[s], a.cap));
    if (b1 > b0 && x.hi > 0) {
      x.tok0 = ba_qs(a, b0);
      x.ntok = max(0, ba_qs(a, b1) - x.tok0);
    }
    x.table = max(0, min(b0, a.B - 1));
  } else {
    x.tok0 = ba_qs(a, s);
    x.ntok = max(0, ba_qs(a, s + 1) - x.tok0);
    const int T = max(0, a.seq_lens[s]);
    x.past = T - x.ntok;
    x.lo = ba_shared(a, s);
    x.hi = min(T, a.cap);
    x.prefix = a.prefix_lens ? a.prefix_lens[s] : 0;
    x.table = s;
  }
  return x;
}

// Lays line L out: the items of every segment, their places, and the item that each wave's
// piece begins in.
template <int L>
__device__ __forceinline__ void ba_lay_out(const BaArgs& a, int32_t* base_s, int64_t* start_s, int64_t* part) {
  const BaLine& ln = a.line[L];
  const int tid = threadIdx.x, R = ln.rows;
  const int nseg = L == 1 ? a.n_groups : a.B;
  // first items of the segments
  int64_t run = 0;
  BaSeg mine{};  // of segment tid, for the common step of one item per segment
  for (int s0 = 0; s0 < nseg; s0 += kPrepThreads) {
    const int s = s0 + tid;
    int64_t n = 0, all;
    if (s < nseg) {
      const BaSeg x = ba_segment<L>(a, s);
      n = ba_div((int64_t)x.ntok * a.G + R - 1, R);
      if (s0 == 0) mine = x;
    }
    const int64_t at = prep_scan(n, part, &all);
    if (s < nseg) base_s[s] = ln.seg_item[s] = (int)min<int64_t>(run + at, INT_MAX);
    run += all;
  }
  if (tid == 0) base_s[nseg] = ln.seg_item[nseg] = (int)min<int64_t>(run, INT_MAX);
  __syncthreads();
  // (starts that do not ascend could make more items than there is room for)
  const int n_items = min(base_s[nseg], ln.max_items);
  int64_t place = 0;
  int most = 0;  // tiles of an item
  for (int i0 = 0; i0 < n_items; i0 += kPrepThreads) {
    const int i = i0 + tid;
    int64_t cost = 0, all;
    BaItem it{};
    if (i < n_items) {
      const bool own = i < kPrepThreads && i < nseg && base_s[i] == i && base_s[i + 1] == i + 1;
      const int s = own ? i : ba_last(nseg, i, [&](int k) { return base_s[k]; });
      const BaSeg x = own ? mine : ba_segment<L>(a, s);
      const int64_t row0 = (int64_t)(i - base_s[s]) * R;
      it.tok0 = x.tok0;
      it.row0 = (int)row0;
      it.nrows = x.ntok * a.G;
      it.table = x.table;
      it.lo = x.lo;
      it.hi = x.hi;
      int64_t lo = x.lo, hi = x.hi;
      if (L == 0) {
        const int i0t = (int)ba_div(row0, a.G), i1t = min(x.ntok - 1, (int)ba_div(row0 + R - 1, a.G));
        hi = min<int64_t>(hi, max<int64_t>((int64_t)x.past + i1t + 1, x.prefix));
        if (a.window > 0) lo = max<int64_t>(lo, (int64_t)x.past + i0t + 1 - a.window);
        if (a.token_starts && hi > lo) {
          int first = INT_MAX;
          for (int t = i0t; t <= i1t; ++t) first = min(first, a.token_starts[x.tok0 + t]);
          lo = max<int64_t>(lo, first);
        }
      }
      it.t0 = hi > lo ? (int)(lo >> 6) : 0;
      it.nt = hi > lo ? (int)((hi + 63) >> 6) - it.t0 : 0;
      cost = (int64_t)(it.nt + kBaOver) * a.hkv;
      most = max(most, it.nt);
    }
    const int64_t at = prep_scan(cost, part, &all);
    if (i < n_items) {
      it.start = place + at;
      ln.items[i] = it;
      if (i < kPrepStarts) start_s[i] = it.start;
    }
    place += all;
  }
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) most = max(most, __shfl_xor(most, o, 64));
  __syncthreads();
  if ((tid & 63) == 0) part[tid >> 6] = most;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kPrepWaves; ++w) most = max(most, (int)part[w]);
  // Equal pieces, of two tiles at least: a single one would double what is to be joined.  An (item,
  // head) of n tiles in k pieces costs its waves about 0.6 us for each of n / k tiles, and those
  // who join it 0.01 us for each of k pieces: the sum is least at about sqrt(n / 64) tiles a piece
  // (one token of 8 heads over 524288: 18 + 11 us where two tiles a piece took 14 + 14).
  const int64_t least = max(2, (int)ceilf(sqrtf((float)most * (1.f / kBaBalance))));
  const int64_t chunk = max<int64_t>(least, ba_div(place + ln.waves - 1, ln.waves));
  if (tid == 0) *ln.head = BaHead{chunk, place, n_items, (int)ba_div(place + chunk - 1, chunk)};
  // The item that each wave's piece begins in: a wave per item fills its waves' entries, or,
  // where items abound, each entry searches for its own.
  if (n_items <= 8 * kPrepWaves) {
    __syncthreads();
    for (int i = tid >> 6; i < n_items; i += kPrepWaves) {
      const int64_t from = start_s[i], to = i + 1 < n_items ? start_s[i + 1] : place;
      const int w1 = (int)ba_div(to + chunk - 1, chunk);
      for (int w = (int)ba_div(from + chunk - 1, chunk) + (tid & 63); w < w1; w += 64) ln.work[w] = i;
    }
    for (int w = (int)ba_div(place + chunk - 1, chunk) + tid; w < ln.waves; w += kPrepThreads) ln.work[w] = -1;
    return;
  }
  auto start_of = [&](int i) { return n_items <= kPrepStarts ? start_s[i] : ln.items[i].start; };
  __syncthreads();
  for (int w = tid; w < ln.waves; w += kPrepThreads) {
    const int64_t p = w * chunk;
    int lo = 0, hi = n_items;
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (start_of(mid) <= p) lo = mid;
      else hi = mid;
    }
    ln.work[w] = p < place ? lo : -1;
  }
}

__device__ __forceinline__ uint32_t ba_pack(_Float16 lo, _Float16 hi) {
  typedef _Float16 h2_t __attribute__((ext_vector_type(2)));
  return __builtin_bit_cast(uint32_t, (h2_t){lo, hi});
}

// The exponent e of amax = m 2^e, m in [0.5, 1) (0 for 0, inf or NaN).
__device__ __forceinline__ int ba_exponent(float amax) {
  int e = 0;
  if (amax > 0.f && amax < INFINITY) frexpf(amax, &e);
  return e;
}

// Entry `e` of the tables, for centroids of exponents ke and ve.
__device__ __forceinline__ BaEntry ba_entry(const BaArgs& a, int vbits, int e, int ke, int ve) {
  BaEntry x{};
  const float ksc = ldexpf(1.f, -ke), vsc = ldexpf(1.f, -ve);
  auto split = [](float u, float v, uint32_t& hi, uint32_t& lo) {
    const _Float16 hu = (_Float16)u, hv = (_Float16)v;
    hi = ba_pack(hu, hv);
    lo = ba_pack((_Float16)(u - (float)hu), (_Float16)(v - (float)hv));
  };
  split(a.kcen[e >> 4] * ksc, a.kcen[e & 15] * ksc, x.khi, x.klo);
  const int mask = (1 << vbits) - 1;
  // a byte's four tokens (2 bits), or a pair (3 bits: its top two bits belong to another dim)
  split(a.vcen[e & mask] * vsc, a.vcen[(e >> vbits) & mask] * vsc, x.vhi[0], x.vlo[0]);
  if (vbits == 2) split(a.vcen[(e >> 4) & 3] * vsc, a.vcen[(e >> 6) & 3] * vsc, x.vhi[1], x.vlo[1]);
  x.vsc_inv = ldexpf(1.f, ve);
  return x;
}

// The tables' entries and R_v's operands (one workgroup).
__device__ __forceinline__ void ba_make_tables(const BaArgs& a, int vbits) {
  const int tid = threadIdx.x, lane = tid & 63;
  const int ke = ba_exponent(wave_max(lane < 16 ? fabsf(a.kcen[lane]) : 0.f));
  const int ve = ba_exponent(wave_max(lane < (1 << vbits) ? fabsf(a.vcen[lane]) : 0.f));
  if (tid < 256) a.entries[tid] = ba_entry(a, vbits, tid, ke, ve);
  const int c = lane & 15, g = lane >> 4, ob = tid >> 7, s = tid >> 6 & 1;
  ba_v8h hi, lo;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float v = a.vrot[(16 * (2 * s + (i >> 2)) + 4 * g + (i & 3)) * a.vrot_row + (16 * ob + c) * a.vrot_col];
    hi[i] = (_Float16)v;
    lo[i] = (_Float16)(v - (float)hi[i]);
  }
  static_assert(kPrepThreads == 512, "a thread per lane of the eight operands");
  reinterpret_cast<ba_v8h*>(a.vrot16)[tid] = hi;
  reinterpret_cast<ba_v8h*>(a.vrot16)[512 + tid] = lo;
}

// The position range of token t (see BaToken).
__device__ __forceinline__ void ba_find_token(const BaArgs& a, int t) {
  BaToken x{0, 0, 0, a.B};
  if (a.B > 0 && t >= ba_qs(a, 0) && t < ba_qs(a, a.B)) {
    // token t of a step of single tokens belongs to sequence t
    const int b = t < a.B && ba_qs(a, t) <= t && ba_qs(a, t + 1) > t
                      ? t : ba_last(a.B, t, [&](int i) { return ba_qs(a, i); });
    const int q0 = ba_qs(a, b), T = max(0, a.seq_lens[b]);
    const int64_t p = (int64_t)T - (ba_qs(a, b + 1) - q0) + (t - q0);
    int64_t lo = 0;
    if (a.window > 0) lo = max<int64_t>(lo, p + 1 - a.window);
    if (a.token_starts) lo = max<int64_t>(lo, a.token_starts[t]);
    x.lo = (int)lo;
    x.hi = (int)min<int64_t>(min(T, a.cap), max<int64_t>(p + 1, a.prefix_lens ? a.prefix_lens[b] : 0));
    x.pos = (int)p;
    x.seq = b;
  }
  a.tokens[t] = x;
}

// Workgroups 0 .. n_lines - 1 lay the lines out, the next makes the tables, the others rotate
// 16 rows (a token's head each) a wave and round: Qrot = q R_k^T qscale, scaled by a power of
// two into [2^(kBaQueryTop - 1), 2^kBaQueryTop) and split into fp16 hi (and lo) parts.  Lane (c, g) ends with dims 16 g ..
// 16 g + 15 of row c, the order in which its key bytes come: output 4 k + r of product mb is
// dim 16 k + 4 mb + r.
//   float32 queries: v_mfma_f32_16x16x4f32, 64 products of 8 passes a round.
//   16-bit queries: v_mfma_f32_16x16x32 on the queries as they are; R_k, held in registers over
//   the rounds, in three bfloat16 or two float16 parts (times 2^10: none is subnormal), which
//   carry 24 and 22 bits: 24 or 16 products of 4 passes.
template <int DT>
__device__ __forceinline__ void ba_rotate_rows(const BaArgs& a, int64_t blk, int64_t n_blks, float* rk_s) {
#pragma clang fp contract(off)
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int c = lane & 15, g = lane >> 4;
  const int64_t n_rows = (int64_t)a.n_tokens * a.hq;
  // R_k through LDS, [64][68]: read along its memory whichever its order, used by rows
  {
    const int at = 8 * tid;
    const ba_v4f x0 = *reinterpret_cast<const ba_v4f*>(a.krot + at), x1 = *reinterpret_cast<const ba_v4f*>(a.krot + at + 4);
    const int along = at & 63, across = at >> 6;
    if (a.krot_col == 1) {
      *reinterpret_cast<ba_v4f*>(rk_s + across * 68 + along) = x0;
      *reinterpret_cast<ba_v4f*>(rk_s + across * 68 + along + 4) = x1;
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        rk_s[(along + i) * 68 + across] = x0[i];
        rk_s[(along + 4 + i) * 68 + across] = x1[i];
      }
    }
  }
  const int ke = ba_exponent(wave_max(lane < 16 ? fabsf(a.kcen[lane]) : 0.f));
  __syncthreads();
  constexpr int PARTS = DT == TQ_BF16 ? 3 : 2;
  typedef __bf16 v8b __attribute__((ext_vector_type(8)));
  using v8 = std::conditional_t<DT == TQ_BF16, v8b, ba_v8h>;
  using elem = std::conditional_t<DT == TQ_BF16, __bf16, _Float16>;
  constexpr float kUp = DT == TQ_F16 ? 1024.f : 1.f;
  v8 part[DT == TQ_F32 ? 1 : PARTS][4][2];
  if constexpr (DT != TQ_F32) {
#pragma unroll
    for (int mb = 0; mb < 4; ++mb)
#pragma unroll
      for (int s = 0; s < 2; ++s)
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          float v = kUp * rk_s[(16 * (c >> 2) + 4 * mb + (c & 3)) * 68 + 32 * s + 8 * g + i];
#pragma unroll
          for (int p = 0; p < PARTS; ++p) {
            const elem x = (elem)v;
            part[p][mb][s][i] = x;
            v -= (float)x;
          }
        }
  }
  for (int64_t r0 = (blk * kPrepWaves + wave) * 16; r0 < n_rows; r0 += n_blks * kPrepWaves * 16) {
    const int64_t row = min(r0 + c, n_rows - 1);
    const int64_t qt = ba_div(row, a.hq), qo = qt * a.q_stride + (row - qt * a.hq) * 64;
    ba_v4f d[4];
    if constexpr (DT == TQ_F32) {
      float qv[16];
      const ba_v4f* src = reinterpret_cast<const ba_v4f*>(static_cast<const float*>(a.q) + qo + 16 * g);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const ba_v4f v = src[i];
        qv[4 * i] = v.x; qv[4 * i + 1] = v.y; qv[4 * i + 2] = v.z; qv[4 * i + 3] = v.w;
      }
#pragma unroll
      for (int mb = 0; mb < 4; ++mb) {
        float rk[16];
#pragma unroll
        for (int i = 0; i < 16; ++i)
          rk[i] = rk_s[(16 * (c >> 2) + 4 * mb + (c & 3)) * 68 + 16 * g + i];
        d[mb] = (ba_v4f){0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int i = 0; i < 16; ++i) d[mb] = __builtin_amdgcn_mfma_f32_16x16x4f32(rk[i], qv[i], d[mb], 0, 0, 0);
      }
    } else {
      v8 q8[2];
#pragma unroll
      for (int s = 0; s < 2; ++s)
        q8[s] = *reinterpret_cast<const v8*>(static_cast<const uint16_t*>(a.q) + qo + 32 * s + 8 * g);
#pragma unroll
      for (int mb = 0; mb < 4; ++mb) {
        d[mb] = (ba_v4f){0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int p = PARTS - 1; p >= 0; --p)  // the small parts first
#pragma unroll
          for (int s = 0; s < 2; ++s) {
            if constexpr (DT == TQ_BF16) d[mb] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(part[p][mb][s], q8[s], d[mb], 0, 0, 0);
            else d[mb] = __builtin_amdgcn_mfma_f32_16x16x32_f16(part[p][mb][s], q8[s], d[mb], 0, 0, 0);
          }
      }
    }
    float qm = 0.f;
#pragma unroll
    for (int mb = 0; mb < 4; ++mb)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        d[mb][r] *= a.qscale * (1.f / kUp);
        qm = fmaxf(qm, fabsf(d[mb][r]));
      }
    qm = fmaxf(qm, __shfl_xor(qm, 16, 64));
    qm = fmaxf(qm, __shfl_xor(qm, 32, 64));
    const int e = max(ba_exponent(qm), -110);  // (2^(14 - e) is finite, its inverse normal)
    const float qsc = ldexpf(1.f, kBaQueryTop - e);
    ba_v8h hi[2], lo[2];
#pragma unroll
    for (int s = 0; s < 2; ++s)
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float v = d[2 * s + (i >> 2)][i & 3] * qsc;
        hi[s][i] = (_Float16)v;
        lo[s][i] = (_Float16)(v - (float)hi[s][i]);
      }
    if (r0 + c < n_rows) {
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        *reinterpret_cast<ba_v8h*>(a.qhi + row * 64 + 16 * g + 8 * s) = hi[s];
        if constexpr (DT != TQ_BF16) *reinterpret_cast<ba_v8h*>(a.qlo + row * 64 + 16 * g + 8 * s) = lo[s];
      }
      if (g == 0) a.qexp[row] = qm > 0.f ? e - kBaQueryTop + ke : -1000;  // (zeros scale no other row)
    }
  }
}

template <int DT>
__global__ __launch_bounds__(kPrepThreads) void batch_prep_kernel(BaArgs a, int n_lines, int vbits) {
  __shared__ int32_t base_s[kBaMaxSegs + 2];
  __shared__ int64_t start_s[kPrepStarts];
  __shared__ int64_t part[kPrepWaves];
  __shared__ __attribute__((aligned(16))) float rk_s[64 * 68];
  if ((int)blockIdx.x < n_lines) {
    if (blockIdx.x == 0) ba_lay_out<0>(a, base_s, start_s, part);
    else ba_lay_out<1>(a, base_s, start_s, part);
    return;
  }
  const int64_t blk = (int64_t)blockIdx.x - n_lines - 1, n_blks = (int64_t)gridDim.x - n_lines - 1;
  if (blk < 0) {
    ba_make_tables(a, vbits);
    return;
  }
  for (int64_t t = blk * kPrepThreads + threadIdx.x; t < a.n_tokens; t += n_blks * kPrepThreads) ba_find_token(a, (int)t);
  ba_rotate_rows<DT>(a, blk, n_blks, rk_s);
}

// ------------------------------------------------------------------------------- joining

// Where one line left a row's sums: by row (one source), or in the slots of `count` waves
// from w0 on.
struct BaFrom {
  int64_t w0;
  int count, row;  // the row in its item
  bool by_row;
};

__device__ __forceinline__ BaFrom ba_from(const BaArgs& a, const BaLine& ln, int seg, int64_t seg_row, int h) {
  BaFrom f{};
  const int n_items = ln.head->n_items;
  if (n_items <= 0 || seg_row < 0) return f;
  const BaItem it = ln.items[max(0, min(ln.seg_item[seg] + (int)ba_div(seg_row, ln.rows), n_items - 1))];
  const int64_t chunk = ln.head->chunk;
  const int cost = it.nt + kBaOver;
  const int64_t start = it.start + (int64_t)h * cost;
  f.row = (int)(seg_row - ba_div(seg_row, ln.rows) * ln.rows);
  // the waves that the first and the last tile fall to
  f.w0 = ba_div(start + kBaOver, chunk);
  const int64_t w1 = ba_div(start + cost - 1, chunk);
  f.by_row = it.nt == 0 || f.w0 == w1;
  f.count = f.by_row ? 1 : (int)(w1 - f.w0) + 1;
  return f;
}

constexpr int kJoinAhead = 4;   // sources a wave asks for at once
constexpr int kTailBlocks = 32;

// ROWS = 16 rows (a token's head each) per workgroup, lane (c, g) dims 16 nb + 4 g .. of row c.
// WAVES waves take a row's sources in turn and join theirs, then share the rotation of the whole
// back by R_v.  A source is 264 bytes of a row; latency bounds a few of them (5 us with the launch).
// ROWS = 1: a workgroup per row, whose columns c take sources in turn too: a CU reads what others
// wrote at about 40 GB/s, so few rows of many pieces need more CUs.
//   kJoinRows: any 16 neighbouring rows; a row's sources are its sequence's line's and, with
//   groups, its group's.
//   Where waves write the results of whole items themselves, the last kTailBlocks workgroups
//   write the rows behind the last sequence, and
//   kJoinItems: workgroup (item, head, j) joins group (ROWS = 1: row) j of the (item, head) if
//   it was cut;
//   kJoinBorders: workgroup (w, j) joins group j of the (item, head) that the border before
//   wave w's piece cuts, if it is that one's first border.
enum { kJoinRows, kJoinItems, kJoinBorders };
template <int BY, int WAVES, int ROWS>
__global__ __launch_bounds__(64 * WAVES) void batch_join_kernel(BaArgs a) {
#pragma clang fp contract(off)
  __shared__ __attribute__((aligned(16))) float sums_s[WAVES][16][68];
  __shared__ float stat_s[WAVES][16][2];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int c = lane & 15, g = lane >> 4;
  const BaLine& ln0 = a.line[0];
  int tok, qh;
  int64_t rowid;
  bool live, known = true;  // the lane's row exists; it belongs to a sequence
  BaFrom s{}, p{};          // sources in lines 0 and 1
  if constexpr (BY != kJoinRows) {
    const int groups = ln0.rows / ROWS;
    const int u = (int)(blockIdx.x / (unsigned)groups), j = (int)(blockIdx.x % (unsigned)groups);
    const unsigned tail = gridDim.x - kTailBlocks;
    if (blockIdx.x >= tail) {
      const int first = a.B > 0 ? ba_qs(a, a.B) : 0, head = a.B > 0 ? ba_qs(a, 0) : 0;
      const int64_t n = (int64_t)(a.n_tokens - first + head) * a.hq;
      constexpr int kRows = 4 * WAVES;
      for (int64_t i = (int64_t)(blockIdx.x - tail) * kRows + (tid >> 4); i < n;
           i += kTailBlocks * kRows) {
        const int t = (int)ba_div(i, a.hq);
        tok = t < head ? t : first + t - head;
        qh = (int)(i - (int64_t)t * a.hq);
        if (a.zero_tail) ba_store(a, tok, qh, 4 * c, (ba_v4f){0.f, 0.f, 0.f, 0.f});
        if (a.lse && c == 0) a.lse[(int64_t)tok * a.hq + qh] = -INFINITY;
      }
      return;
    }
    const BaHead hd = *ln0.head;
    int i, h;
    if constexpr (BY == kJoinItems) {
      i = u / a.hkv;
      h = u - i * a.hkv;
      if (i >= hd.n_items) return;
    } else {
      if ((u + 1) * hd.chunk >= hd.total) return;
      i = ln0.work[u + 1];
    }
    const BaItem it = ln0.items[i];
    const int64_t cost = it.nt + kBaOver;
    if constexpr (BY == kJoinBorders) h = (int)ba_div((u + 1) * hd.chunk - it.start, cost);
    const int64_t start = it.start + h * cost;
    s.w0 = ba_div(start + kBaOver, hd.chunk);
    const int64_t w1 = ba_div(start + cost - 1, hd.chunk);
    if (s.w0 == w1 || it.nt == 0 || it.row0 + ROWS * j >= it.nrows || (BY == kJoinBorders && u != (int)s.w0)) return;
    s.count = (int)(w1 - s.w0) + 1;
    s.row = ROWS * j + (ROWS > 1 ? c : 0);
    live = it.row0 + s.row < it.nrows;
    const int row = min(it.row0 + s.row, it.nrows - 1), ti = row / a.G;
    tok = it.tok0 + ti;
    qh = h * a.G + (row - ti * a.G);
    rowid = (int64_t)tok * a.hq + qh;
  } else {
    const int64_t n_rows = (int64_t)a.n_tokens * a.hq, r0 = (int64_t)blockIdx.x * ROWS;
    rowid = min(r0 + (ROWS > 1 ? c : 0), n_rows - 1);
    live = r0 + (ROWS > 1 ? c : 0) < n_rows;
    tok = (int)ba_div(rowid, a.hq);
    qh = (int)(rowid - (int64_t)tok * a.hq);
  }
  // R_v's operands of this wave's dims (wave ob: 16 ob ..; one wave: all), wanted last
  constexpr int OBS = 4 / WAVES;
  ba_v8h rv[OBS][2][2];
  auto load_rv = [&] {
#pragma unroll
    for (int ob = 0; ob < OBS; ++ob)
#pragma unroll
      for (int part = 0; part < 2; ++part)
#pragma unroll
        for (int k = 0; k < 2; ++k)
          rv[ob][part][k] = reinterpret_cast<const ba_v8h*>(a.vrot16)[(part * 8 + (wave * OBS + ob) * 2 + k) * 64 + lane];
  };
  if constexpr (WAVES > 1) load_rv();
  if constexpr (BY == kJoinRows) {
    const int h = qh / a.G, gq = qh - h * a.G;
    const BaToken t = a.tokens[tok];
    known = t.seq < a.B;
    if (known) {
      s = ba_from(a, ln0, t.seq, (int64_t)(tok - ba_qs(a, t.seq)) * a.G + gq, h);
      if (a.n_groups > 0) {
        const int gi = ba_last(a.n_groups, t.seq, [&](int i) { return a.group_start[i]; });
        const int b0 = a.group_start[gi], b1 = min(a.group_start[gi + 1], a.B);
        if (b0 >= 0 && t.seq >= b0 && t.seq < b1 && a.shared[gi] > 0 && a.cap > 0)
          p = ba_from(a, a.line[1], gi, (int64_t)(tok - ba_qs(a, b0)) * a.G + gq, h);
      }
    }
  }
  const int ns = s.count, np = p.count;
  int most = ns + np;
#pragma unroll
  for (int o = 8; o >= 1; o >>= 1) most = max(most, __shfl_xor(most, o, 64));
  most = __builtin_amdgcn_readfirstlane(most);

  struct Source {
    float m, l;
    ba_v4f v[4];
  };
  // source i of the lane's row (behind its last: nothing)
  auto load = [&](int i, Source& x) {
    const bool mine = i < ns, any = i < ns + np;
    const BaFrom& f = mine ? s : p;
    const BaLine& ln = BY != kJoinRows || mine || !any ? ln0 : a.line[1];
    const int k = !any ? 0 : mine ? i : i - ns;
    // the wave with the item's first tile kept it in slot 1
    const float* slot = ln.slots + (any ? (f.w0 + k) * 2 + (k == 0) : 0) * ba_slot_floats(ln.rows);
    const bool by_row = BY == kJoinRows && any && f.by_row;
    const int row = any ? f.row : 0;
    const float* sums = by_row ? ln.row_sums + rowid * 64 : slot + row * 64;
    const float* st = by_row ? ln.row_stats + rowid * 2 : slot + ln.rows * 64 + row * 2;
    x.m = st[0];
    x.l = st[1];
#pragma unroll
    for (int nb = 0; nb < 4; ++nb) x.v[nb] = *reinterpret_cast<const ba_v4f*>(sums + 16 * nb + 4 * g);
    if (!any) {  // (what was read may be NaN)
      x.m = -INFINITY;
      x.l = 0.f;
#pragma unroll
      for (int nb = 0; nb < 4; ++nb) x.v[nb] = (ba_v4f){0.f, 0.f, 0.f, 0.f};
    }
  };
  float m = -INFINITY, l = 0.f;
  ba_v4f o4[4];
#pragma unroll
  for (int nb = 0; nb < 4; ++nb) o4[nb] = (ba_v4f){0.f, 0.f, 0.f, 0.f};
  auto add = [&](const Source& x) {
    const float mn = fmaxf(m, x.m), ms = mn == -INFINITY ? 0.f : mn;
    const float fa = __builtin_amdgcn_exp2f(m - ms), fb = __builtin_amdgcn_exp2f(x.m - ms);
    m = mn;
    l = l * fa + x.l * fb;
#pragma unroll
    for (int nb = 0; nb < 4; ++nb) o4[nb] = o4[nb] * fa + x.v[nb] * fb;
  };
  constexpr int STEP = WAVES * (16 / ROWS);  // sources taken at once
  const int first = ROWS > 1 ? wave : 16 * wave + c;
  if (most <= STEP) {
    if (first < most) {
      Source x;
      load(first, x);
      add(x);
    }
  } else {
    constexpr int AHEAD = WAVES > 1 ? kJoinAhead : 2;
    for (int i = 0; i < most; i += AHEAD * STEP) {
      Source x[AHEAD];
#pragma unroll
      for (int u = 0; u < AHEAD; ++u) load(i + first + u * STEP, x[u]);
#pragma unroll
      for (int u = 0; u < AHEAD; ++u) add(x[u]);
    }
  }
  if constexpr (ROWS == 1) {  // over the columns
    float mn = m;
#pragma unroll
    for (int o = 1; o < 16; o <<= 1) mn = fmaxf(mn, __shfl_xor(mn, o, 64));
    const float f = __builtin_amdgcn_exp2f(m - (mn == -INFINITY ? 0.f : mn));
    m = mn;
    l *= f;
#pragma unroll
    for (int nb = 0; nb < 4; ++nb) o4[nb] *= f;
#pragma unroll
    for (int o = 1; o < 16; o <<= 1) {
      l += __shfl_xor(l, o, 64);
#pragma unroll
      for (int nb = 0; nb < 4; ++nb)
#pragma unroll
        for (int r = 0; r < 4; ++r) o4[nb][r] += __shfl_xor(o4[nb][r], o, 64);
    }
  }
  if constexpr (WAVES > 1) {
#pragma unroll
    for (int nb = 0; nb < 4; ++nb) *reinterpret_cast<ba_v4f*>(&sums_s[wave][c][16 * nb + 4 * g]) = o4[nb];
    if (g == 0) {
      stat_s[wave][c][0] = m;
      stat_s[wave][c][1] = l;
    }
    __syncthreads();
    float f[WAVES];
    m = -INFINITY;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) m = fmaxf(m, stat_s[w][c][0]);
    const float ms = m == -INFINITY ? 0.f : m;
    l = 0.f;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) {
      f[w] = __builtin_amdgcn_exp2f(stat_s[w][c][0] - ms);
      l += stat_s[w][c][1] * f[w];
    }
#pragma unroll
    for (int nb = 0; nb < 4; ++nb) {
      o4[nb] = (ba_v4f){0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int w = 0; w < WAVES; ++w) o4[nb] += *reinterpret_cast<const ba_v4f*>(&sums_s[w][c][16 * nb + 4 * g]) * f[w];
    }
  } else {
    load_rv();
  }
  // ba_rotate_back for this wave's dims, into fp16's range by a power of two of the row
  const float inv = l == 0.f ? 0.f : 1.f / l;
  float xm = 0.f;
#pragma unroll
  for (int nb = 0; nb < 4; ++nb) {
    o4[nb] *= inv;
#pragma unroll
    for (int r = 0; r < 4; ++r) xm = fmaxf(xm, fabsf(o4[nb][r]));
  }
  xm = fmaxf(xm, __shfl_xor(xm, 16, 64));
  xm = fmaxf(xm, __shfl_xor(xm, 32, 64));
  const int e = max(ba_exponent(xm), -122);  // (2^(4 - e) is finite, its inverse normal)
  const float up = ldexpf(1.f, 4 - e), down = ldexpf(1.f, e - 4);
  ba_v8h hi[2], lo[2];
#pragma unroll
  for (int k = 0; k < 2; ++k)
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      _Float16 hv, lv;
      split_f16(o4[2 * k + (u >> 2)][u & 3] * up, hv, lv);
      hi[k][u] = hv;
      lo[k][u] = lv;
    }
  mfma_operand_fence(hi[0], hi[1], lo[0], lo[1]);
  ba_v4f acc[OBS];
#pragma unroll
  for (int ob = 0; ob < OBS; ++ob) {
    acc[ob] = (ba_v4f){0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      acc[ob] = __builtin_amdgcn_mfma_f32_16x16x32_f16(rv[ob][1][k], hi[k], acc[ob], 0, 0, 0);
      acc[ob] = __builtin_amdgcn_mfma_f32_16x16x32_f16(rv[ob][0][k], lo[k], acc[ob], 0, 0, 0);
      acc[ob] = __builtin_amdgcn_mfma_f32_16x16x32_f16(rv[ob][0][k], hi[k], acc[ob], 0, 0, 0);
    }
    acc[ob] *= down;
  }
  if (!live || (ROWS == 1 && c > 0)) return;
  if (known || a.zero_tail)
#pragma unroll
    for (int ob = 0; ob < OBS; ++ob) ba_store(a, tok, qh, 16 * (wave * OBS + ob) + 4 * g, acc[ob]);
  if (a.lse && wave == 0 && g == 0) a.lse[rowid] = ba_lse(m, l);
}

// --------------------------------------------------------------------------------- plans

// Which kernels a call runs, and its workspace.
struct BaPlan {
  bool prec, pair;
  bool direct;           // waves write the results of whole items
  int rw[2], groups[2];  // per line: rows of a group of columns, groups
  int64_t items[2];
  unsigned grid;
  int64_t segs[2];
};

BaPlan ba_plan(tq_dtype q_dtype, int64_t n, int hq, int hkv, int64_t B, int64_t n_groups, int64_t capacity) {
  BaPlan p{};
  p.prec = q_dtype != TQ_BF16;
  const int G = hq / hkv;
  const int64_t rows = n * G, cus = device_cu_count();
  p.pair = n_groups > 0;
  p.segs[0] = B;
  p.segs[1] = n_groups;
  for (int l = 0; l < (n_groups > 0 ? 2 : 1); ++l) {
    // A group of columns as wide as a segment's rows are on average: single tokens of few heads
    // use 4 or 8 of the 16 columns; rows beyond 16 share each tile's lookups.
    // (rounded: a few rows of padding behind single tokens do not widen them)
    const int64_t segs = std::max<int64_t>(l ? n_groups : B, 1);
    const int64_t avg = std::max<int64_t>(1, (n + segs / 2) / segs) * G;
    p.rw[l] = l == 1 || avg > 8 ? 16 : avg <= 4 ? 4 : 8;
    p.groups[l] = l == 1 || avg > 16 ? ba_groups(p.prec, p.pair) : 1;  // (groups hold many rows)
    const int R = p.rw[l] * p.groups[l];
    p.items[l] = rows / R + p.segs[l];
    // one workgroup per CU, fewer where even one-tile pieces would not fill them
    const int64_t pieces = p.items[l] * hkv * (capacity / 64 + 1 + kBaOver);
    p.grid = std::max(p.grid, (unsigned)std::max<int64_t>(1, std::min(cus, pieces)));
  }
  p.direct = !p.pair && p.groups[0] > 1;
  return p;
}

// Places the workspace's parts from `at` on (null: only counts); the bytes taken.
size_t ba_place(const BaPlan& p, int64_t n, int hq, char* at, BaArgs* a) {
  size_t used = 0;
  auto take = [&](size_t bytes) {
    char* here = at ? at + used : nullptr;
    used += align_up(bytes, 256);
    return here;
  };
  const size_t rows = (size_t)n * hq;
  BaArgs b{};
  b.entries = reinterpret_cast<BaEntry*>(take(256 * sizeof(BaEntry)));
  b.tokens = reinterpret_cast<BaToken*>(take(n * sizeof(BaToken)));
  b.qexp = reinterpret_cast<int32_t*>(take(rows * 4));
  b.qhi = reinterpret_cast<_Float16*>(take(rows * 128));
  b.vrot16 = reinterpret_cast<_Float16*>(take(2 * 4096 * sizeof(_Float16)));
  if (p.prec) b.qlo = reinterpret_cast<_Float16*>(take(rows * 128));
  for (int l = 0; l < 2; ++l) {
    if (l == 1 && !p.pair) continue;
    BaLine& ln = b.line[l];
    ln.waves = (int)p.grid * kBaWaves;
    ln.rows = p.rw[l] * p.groups[l];
    ln.max_items = (int)p.items[l];
    ln.head = reinterpret_cast<BaHead*>(take(sizeof(BaHead)));
    ln.items = reinterpret_cast<BaItem*>(take(p.items[l] * sizeof(BaItem)));
    ln.seg_item = reinterpret_cast<int32_t*>(take((p.segs[l] + 1) * 4));
    ln.work = reinterpret_cast<int32_t*>(take((size_t)ln.waves * 4));
    ln.slots = reinterpret_cast<float*>(take((size_t)ln.waves * 2 * ba_slot_floats(ln.rows) * 4));
    if (p.direct) continue;  // whole items leave results, not sums
    ln.row_sums = reinterpret_cast<float*>(take(rows * 256));
    ln.row_stats = reinterpret_cast<float*>(take(rows * 8));
  }
  if (a) {
    a->entries = b.entries; a->vrot16 = b.vrot16; a->tokens = b.tokens; a->qexp = b.qexp; a->qhi = b.qhi; a->qlo = b.qlo;
    a->line[0] = b.line[0]; a->line[1] = b.line[1];
  }
  return used;
}

template <int VB>
void ba_run_bits(const BaArgs& a, const BaPlan& p, hipStream_t st) {
  const bool wide = (uint64_t)a.num_blocks * a.hkv << a.bs_log2 > 0xFFFFFFFFu / 32;  // key bytes past 32 bits
  if (a.bs_log2 < 6) ba_launch<VB, true>(a, p.pair, wide, p.prec, p.rw[0], p.groups[0], p.grid, st);
  else ba_launch<VB, false>(a, p.pair, wide, p.prec, p.rw[0], p.groups[0], p.grid, st);
}

void ba_run(int vbits, const BaArgs& a, const BaPlan& p, hipStream_t st) {
  if (vbits == 2) ba_run_bits<2>(a, p, st);
  else if (vbits == 3) ba_run_bits<3>(a, p, st);
  else ba_run_bits<4>(a, p, st);
}

template <int BY, int WAVES, int ROWS>
void ba_join_by(const BaArgs& a, int64_t grid, hipStream_t st) {
  hipLaunchKernelGGL((batch_join_kernel<BY, WAVES, ROWS>), dim3((unsigned)grid), dim3(64 * WAVES), 0, st, a);
}

// Few rows, whose pieces may be many, have a workgroup each (one token of 8 heads over 131072: 17.8 ->
// 7.1 us; 48 tokens of 32 heads over 8192 fill the chip with 16 rows each: 6.4 us against 14.2).
// Where waves wrote whole items themselves and the waves are at most four to an (item, head), few
// of those lie in many pieces, and a wave joins each: 15 us for 4096-token prompts where four waves
// took 28, 9.7 against 12.0 for chunks of 512 over 12288.
void ba_join(const BaArgs& a, const BaPlan& p, hipStream_t st) {
  const int64_t pairs = p.items[0] * a.hkv, R = a.line[0].rows;
  const int64_t rows = (int64_t)a.n_tokens * a.hq, most = 2 * device_cu_count();
  if (!a.direct) {
    if (rows <= most) ba_join_by<kJoinRows, 4, 1>(a, rows, st);
    else ba_join_by<kJoinRows, 4, 16>(a, (rows + 15) / 16, st);
  } else if (pairs * 4 >= a.line[0].waves) {
    ba_join_by<kJoinBorders, 1, 16>(a, (a.line[0].waves - 1) * (R / 16) + kTailBlocks, st);
  } else if (rows <= most) {
    ba_join_by<kJoinItems, 4, 1>(a, pairs * R + kTailBlocks, st);
  } else {
    ba_join_by<kJoinItems, 4, 16>(a, pairs * (R / 16) + kTailBlocks, st);
  }
}

}  // namespace
}  // namespace tq

using namespace tq;

extern "C" {

size_t tq_attention_batch_workspace_bytes(tq_dtype q_dtype, int32_t n_tokens, int32_t hq, int32_t hkv,
                                          int32_t n_seqs, int32_t n_groups, int64_t capacity) {
  if (n_tokens <= 0 || hkv < 1 || hq < hkv || hq % hkv || n_seqs < 0 || n_groups < 0 || capacity < 0) return 0;
  return ba_place(ba_plan(q_dtype, n_tokens, hq, hkv, n_seqs, n_groups, capacity), n_tokens, hq, nullptr, nullptr);
}

int tq_attention_batch_paged_dl(const void* q, tq_dtype q_dtype, int32_t n_tokens, int64_t q_stride, int32_t hq,
                                int32_t hkv, int32_t d, const uint8_t* kpairs_pool, const float* knorm_pool,
                                const uint8_t* vtile_pool, const float* vnorm_pool, int64_t num_blocks,
                                int32_t block_size, int32_t vbits, const int32_t* block_tables,
                                int64_t table_stride, int32_t max_blocks, const int32_t* query_start_loc,
                                const int32_t* seq_lens, int32_t n_seqs, const int32_t* group_start_loc,
                                const int32_t* shared_lens, int32_t n_groups, const float* kcentroids,
                                const float* vcentroids, const float* krotation, const float* vrotation,
                                int32_t transposed, float scale, const tq_score_variant* variant, void* out, int64_t out_stride,
                                int32_t zero_tail, float* lse, void* workspace, size_t workspace_bytes,
                                void* stream) {
  TQ_REQUIRE(valid_dtype(q_dtype), "unknown dtype");
  TQ_REQUIRE(d == 64, "decode layout covers head_dim 64, got %d", d);
  TQ_REQUIRE(vbits >= 2 && vbits <= 4, "value tiles hold 2-4 bit codes, got %d", vbits);
  TQ_REQUIRE(hkv >= 1 && hq >= hkv && hq % hkv == 0, "num_heads (%d) must be a multiple of num_kv_heads (%d)", hq,
             hkv);
  int bsl = 0;
  while (bsl < 30 && (1 << bsl) < block_size) ++bsl;
  TQ_REQUIRE(block_size >= 16 && (1 << bsl) == block_size,
             "decode-layout pools need a power-of-two block_size >= 16, got %d", block_size);
  TQ_REQUIRE(n_tokens >= 0 && n_seqs >= 0 && n_groups >= 0 && max_blocks >= 0 && num_blocks >= 0, "bad sizes");
  TQ_REQUIRE(n_seqs <= kBaMaxSegs && n_groups <= kBaMaxSegs, "a call takes at most %d sequences and groups, got %d and %d",
             kBaMaxSegs, n_seqs, n_groups);
  TQ_REQUIRE(num_blocks <= (int64_t)UINT_MAX, "too many blocks");
  TQ_REQUIRE(table_stride >= max_blocks, "table rows of %d entries overlap at a stride of %lld", max_blocks,
             (long long)table_stride);
  const int64_t cap = (int64_t)max_blocks * block_size;
  TQ_REQUIRE(cap <= INT_MAX - 127, "a table's capacity exceeds 2^31 - 128 tokens");
  const int64_t rows = (int64_t)n_tokens * (hq / hkv);
  TQ_REQUIRE(rows <= INT_MAX - 1024, "too many query rows in one call");
  if (n_tokens == 0) return TQ_OK;
  const int64_t row_elems = (int64_t)hq * 64;
  TQ_REQUIRE(q_stride >= row_elems && out_stride >= row_elems, "rows of %lld elements overlap", (long long)row_elems);
  const tq_score_variant none{};
  const tq_score_variant& v = variant ? *variant : none;
  TQ_REQUIRE(v.softcap == 0.f || (v.softcap >= 1e-30f && v.softcap <= 1e30f),
             "softcap must be 0 or in [1e-30, 1e30], got %g", v.softcap);
  TQ_REQUIRE(v.window >= 0, "window must not be negative, got %d", v.window);
  TQ_REQUIRE(q && out && (n_seqs == 0 || (query_start_loc && seq_lens)) && kcentroids && vcentroids && krotation &&
                 vrotation && (n_groups == 0 || (group_start_loc && shared_lens)),
             "null pointer argument");
  TQ_REQUIRE(n_seqs == 0 || max_blocks == 0 || block_tables, "null pointer argument");
  const bool empty = max_blocks == 0 || num_blocks == 0;  // no token is visible
  TQ_REQUIRE(empty || (kpairs_pool && knorm_pool && vtile_pool && vnorm_pool), "null pointer argument");
  TQ_REQUIRE(((reinterpret_cast<uintptr_t>(kpairs_pool) | reinterpret_cast<uintptr_t>(vtile_pool) |
               reinterpret_cast<uintptr_t>(knorm_pool) | reinterpret_cast<uintptr_t>(vnorm_pool) |
               reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(out) |
               reinterpret_cast<uintptr_t>(krotation)) &
              15u) == 0,
             "queries, pools, rotations and output must be 16-byte aligned");
  const size_t esz = dtype_size(q_dtype);
  TQ_REQUIRE(q_stride * esz % 16 == 0 && out_stride * esz % 16 == 0, "token strides must be multiples of 16 bytes");
  const BaPlan p = ba_plan(q_dtype, n_tokens, hq, hkv, n_seqs, n_groups, cap);
  TQ_REQUIRE(p.items[0] <= INT_MAX && p.items[1] <= INT_MAX && (int64_t)n_tokens * hq <= (int64_t)INT_MAX * 16,
             "too many query rows in one call");
  BaArgs a{};
  const size_t need = ba_place(p, n_tokens, hq, static_cast<char*>(workspace), &a);
  TQ_REQUIRE(workspace && workspace_bytes >= need, "workspace too small: need %zu bytes", need);
  TQ_REQUIRE((reinterpret_cast<uintptr_t>(workspace) & 15u) == 0, "workspace must be 16-byte aligned");
  a.q = q; a.q_stride = q_stride; a.q_dt = (int)q_dtype;
  a.n_tokens = n_tokens; a.hq = hq; a.hkv = hkv; a.G = hq / hkv; a.B = n_seqs;
  a.query_start = query_start_loc; a.seq_lens = seq_lens;
  a.group_start = n_groups ? group_start_loc : nullptr; a.shared = shared_lens; a.n_groups = n_groups;
  a.kpairs = kpairs_pool; a.knorms = knorm_pool; a.vtiles = vtile_pool; a.vnorms = vnorm_pool;
  a.block_tables = block_tables; a.table_stride = table_stride;
  a.max_blocks = max_blocks; a.bs_log2 = bsl; a.num_blocks = (uint32_t)num_blocks;
  a.cap = empty ? 0 : (int)cap;
  a.kcen = kcentroids; a.vcen = vcentroids; a.krot = krotation; a.vrot = vrotation;
  a.krot_row = transposed & 1 ? 1 : 64; a.krot_col = transposed & 1 ? 64 : 1;
  a.vrot_row = transposed & 2 ? 1 : 64; a.vrot_col = transposed & 2 ? 64 : 1;
  a.qscale = scale * 1.4426950408889634f;
  if (v.softcap > 0.f) {
    a.cap2 = v.softcap * 1.4426950408889634f;
    a.cap2_inv = 1.f / a.cap2;
  }
  a.slopes = v.alibi_slopes; a.window = v.window; a.prefix_lens = v.prefix_lens; a.token_starts = v.token_starts;
  a.out = out; a.out_stride = out_stride; a.lse = lse; a.zero_tail = zero_tail;
  hipStream_t st = as_stream(stream);
  const int lines = n_groups > 0 ? 2 : 1;
  const int64_t qrows = (int64_t)n_tokens * hq;
  a.direct = p.direct;
  // waves of several rounds share R_k's parts: about two workgroups a CU at the most
  const int64_t rot = std::min<int64_t>((qrows + 16 * kPrepWaves - 1) / (16 * kPrepWaves), 2 * device_cu_count());
  const dim3 prep((unsigned)(lines + 1 + rot)), pthreads(kPrepThreads);
  if (q_dtype == TQ_F32) hipLaunchKernelGGL((batch_prep_kernel<TQ_F32>), prep, pthreads, 0, st, a, lines, vbits);
  else if (q_dtype == TQ_F16) hipLaunchKernelGGL((batch_prep_kernel<TQ_F16>), prep, pthreads, 0, st, a, lines, vbits);
  else hipLaunchKernelGGL((batch_prep_kernel<TQ_BF16>), prep, pthreads, 0, st, a, lines, vbits);
  TQ_LAUNCH_CHECK("batch_prep_kernel");
  ba_run(vbits, a, p, st);
  TQ_LAUNCH_CHECK("batch_attn_kernel");
  ba_join(a, p, st);
  TQ_LAUNCH_CHECK("batch_join_kernel");
  return TQ_OK;
}

}  // extern "C"
