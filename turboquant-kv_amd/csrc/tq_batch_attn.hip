// tq_batch_attn.hip -- entry points of the ragged batch's attention (tq_batch_attn.h): the choice
// of kernels and the workspace, the preparing kernel and the one that joins partial results.

#include "tq_batch_attn.h"

#include <algorithm>

namespace tq {
namespace {

constexpr int kPrepThreads = 512;
constexpr int kPrepWaves = kPrepThreads / 64;
constexpr int kPrepStarts = 2048;  // items' places kept in LDS

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
    }
    const int64_t at = prep_scan(cost, part, &all);
    if (i < n_items) {
      it.start = place + at;
      ln.items[i] = it;
      if (i < kPrepStarts) start_s[i] = it.start;
    }
    place += all;
  }
  // Equal pieces, of two tiles at least: a single one would double what is to be joined.
  const int64_t chunk = max<int64_t>(2, ba_div(place + ln.waves - 1, ln.waves));
  if (tid == 0) *ln.head = BaHead{chunk, place, n_items, 0};
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
    const int e = ba_exponent(qm);
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

constexpr int kJoinWaves = 4;

// 16 rows (a token's head each) per workgroup: a row's sums come from its sequence's line and,
// with groups, from its group's.  The waves take a row's sources in turn, join theirs, then
// wave ob rotates dims 16 ob .. of the whole back by R_v.  A source is 264 bytes of a row;
// latency bounds it (a few microseconds).
__global__ __launch_bounds__(64 * kJoinWaves) void batch_join_kernel(BaArgs a) {
#pragma clang fp contract(off)
  __shared__ __attribute__((aligned(16))) float sums_s[kJoinWaves][16][68];
  __shared__ float stat_s[kJoinWaves][16][2];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int c = lane & 15, g = lane >> 4;
  const int64_t n_rows = (int64_t)a.n_tokens * a.hq, r0 = (int64_t)blockIdx.x * 16;
  const int64_t rowid = min(r0 + c, n_rows - 1);
  const int tok = (int)ba_div(rowid, a.hq), qh = (int)(rowid - (int64_t)tok * a.hq);
  const int h = qh / a.G, gq = qh - h * a.G;
  // R_v's operands of this wave's dims, wanted last
  ba_v8h rv[2][2];
#pragma unroll
  for (int part = 0; part < 2; ++part)
#pragma unroll
    for (int s = 0; s < 2; ++s)
      rv[part][s] = reinterpret_cast<const ba_v8h*>(a.vrot16)[(part * 8 + wave * 2 + s) * 64 + lane];
  const BaToken t = a.tokens[tok];
  BaFrom s{}, p{};
  if (t.seq < a.B) {
    s = ba_from(a, a.line[0], t.seq, (int64_t)(tok - ba_qs(a, t.seq)) * a.G + gq, h);
    if (a.n_groups > 0) {
      const int gi = ba_last(a.n_groups, t.seq, [&](int i) { return a.group_start[i]; });
      const int b0 = a.group_start[gi], b1 = min(a.group_start[gi + 1], a.B);
      if (b0 >= 0 && t.seq >= b0 && t.seq < b1 && a.shared[gi] > 0 && a.cap > 0)
        p = ba_from(a, a.line[1], gi, (int64_t)(tok - ba_qs(a, b0)) * a.G + gq, h);
    }
  }
  const int ns = s.count, np = p.count;
  int most = ns + np;
#pragma unroll
  for (int o = 8; o >= 1; o >>= 1) most = max(most, __shfl_xor(most, o, 64));

  float m = -INFINITY, l = 0.f;
  ba_v4f o4[4];
#pragma unroll
  for (int nb = 0; nb < 4; ++nb) o4[nb] = (ba_v4f){0.f, 0.f, 0.f, 0.f};
  for (int i = wave; i < most; i += kJoinWaves) {
    if (i >= ns + np) continue;
    const bool mine = i < ns;
    const float *sums, *st;
    auto source = [&](const BaLine& ln, const BaFrom& f, int k) {
      // the wave with the item's first tile kept it in slot 1
      const float* slot = ln.slots + ((f.w0 + k) * 2 + (k == 0)) * ba_slot_floats(ln.rows);
      sums = f.by_row ? ln.row_sums + rowid * 64 : slot + f.row * 64;
      st = f.by_row ? ln.row_stats + rowid * 2 : slot + ln.rows * 64 + f.row * 2;
    };
    if (mine) source(a.line[0], s, i);
    else source(a.line[1], p, i - ns);
    const float mi = st[0], li = st[1];
    const float mn = fmaxf(m, mi), ms = mn == -INFINITY ? 0.f : mn;
    const float fa = __builtin_amdgcn_exp2f(m - ms), fb = __builtin_amdgcn_exp2f(mi - ms);
    m = mn;
    l = l * fa + li * fb;
#pragma unroll
    for (int nb = 0; nb < 4; ++nb)
      o4[nb] = o4[nb] * fa + *reinterpret_cast<const ba_v4f*>(sums + 16 * nb + 4 * g) * fb;
  }
#pragma unroll
  for (int nb = 0; nb < 4; ++nb) *reinterpret_cast<ba_v4f*>(&sums_s[wave][c][16 * nb + 4 * g]) = o4[nb];
  if (g == 0) {
    stat_s[wave][c][0] = m;
    stat_s[wave][c][1] = l;
  }
  __syncthreads();
  float M = -INFINITY, L = 0.f, f[kJoinWaves];
#pragma unroll
  for (int w = 0; w < kJoinWaves; ++w) M = fmaxf(M, stat_s[w][c][0]);
  const float Ms = M == -INFINITY ? 0.f : M;
#pragma unroll
  for (int w = 0; w < kJoinWaves; ++w) {
    f[w] = __builtin_amdgcn_exp2f(stat_s[w][c][0] - Ms);
    L += stat_s[w][c][1] * f[w];
  }
  // ba_rotate_back for one ob, into fp16's range by a power of two of the row
  const float inv = L == 0.f ? 0.f : 1.f / L;
  float x[16], xm = 0.f;
#pragma unroll
  for (int nb = 0; nb < 4; ++nb) {
    ba_v4f v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < kJoinWaves; ++w) v += *reinterpret_cast<const ba_v4f*>(&sums_s[w][c][16 * nb + 4 * g]) * f[w];
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      x[4 * nb + r] = v[r] * inv;
      xm = fmaxf(xm, fabsf(x[4 * nb + r]));
    }
  }
  xm = fmaxf(xm, __shfl_xor(xm, 16, 64));
  xm = fmaxf(xm, __shfl_xor(xm, 32, 64));
  const int e = ba_exponent(xm);
  const float up = ldexpf(1.f, 4 - e);
  ba_v8h hi[2], lo[2];
#pragma unroll
  for (int s = 0; s < 2; ++s)
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      _Float16 hv, lv;
      split_f16(x[8 * s + i] * up, hv, lv);
      hi[s][i] = hv;
      lo[s][i] = lv;
    }
  mfma_operand_fence(hi[0], hi[1], lo[0], lo[1]);
  ba_v4f acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int s = 0; s < 2; ++s) {
    acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(rv[1][s], hi[s], acc, 0, 0, 0);
    acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(rv[0][s], lo[s], acc, 0, 0, 0);
    acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(rv[0][s], hi[s], acc, 0, 0, 0);
  }
  acc *= ldexpf(1.f, e - 4);
  if (r0 + c >= n_rows) return;
  if (t.seq < a.B || a.zero_tail) ba_store(a, tok, qh, 16 * wave + 4 * g, acc);
  if (a.lse && wave == 0 && g == 0) a.lse[rowid] = ba_lse(M, L);
}

// Where waves write whole items themselves: workgroup (w, j) joins group j of the (item, head)
// that the border before wave w's piece cuts, if it is that one's first border; the last
// kTailBlocks workgroups write the rows behind the last sequence.  A wave rotates a quarter of the
// dims; all four read the sums of the waves that took a part.
constexpr int kTailBlocks = 32;
template <bool PREC>
__global__ __launch_bounds__(64) void batch_join_cut_kernel(BaArgs a) {
#pragma clang fp contract(off)
  const BaLine& ln = a.line[0];
  const int lane = threadIdx.x, c = lane & 15, g = lane >> 4;
  const int groups = ln.rows / 16;
  const int w = (int)(blockIdx.x / (unsigned)groups) + 1, j = (int)(blockIdx.x % (unsigned)groups);
  if (w >= ln.waves) {
    const int first = a.B > 0 ? ba_qs(a, a.B) : 0, head = a.B > 0 ? ba_qs(a, 0) : 0;
    const int64_t n = (int64_t)(a.n_tokens - first + head) * a.hq;
    for (int64_t i = (int64_t)(blockIdx.x - (unsigned)(groups * (ln.waves - 1))) * 4 + g; i < n; i += kTailBlocks * 4) {
      const int t = (int)ba_div(i, a.hq), qh = (int)(i - (int64_t)t * a.hq);
      const int tok = t < head ? t : first + t - head;
      if (a.zero_tail) ba_store(a, tok, qh, 4 * c, (ba_v4f){0.f, 0.f, 0.f, 0.f});
      if (a.lse && c == 0) a.lse[(int64_t)tok * a.hq + qh] = -INFINITY;
    }
    return;
  }
  const int64_t chunk = ln.head->chunk, p = w * chunk;
  if (p >= ln.head->total) return;
  const BaItem it = ln.items[ln.work[w]];
  const int64_t cost = it.nt + kBaOver;
  const int h = (int)ba_div(p - it.start, cost);
  const int64_t start = it.start + h * cost;
  const int64_t w0 = ba_div(start + kBaOver, chunk), w1 = ba_div(start + cost - 1, chunk);
  const int row = it.row0 + 16 * j + c;
  if (w0 == w1 || it.nt == 0 || w != (int)w0 + 1 || it.row0 + 16 * j >= it.nrows) return;
  float m = -INFINITY, l = 0.f;
  ba_v4f x[4], out[4];
#pragma unroll
  for (int nb = 0; nb < 4; ++nb) x[nb] = (ba_v4f){0.f, 0.f, 0.f, 0.f};
  for (int64_t k = w0; k <= w1; ++k) {
    const float* slot = ln.slots + (k * 2 + (k == w0)) * ba_slot_floats(ln.rows);
    const float* sums = slot + (16 * j + c) * 64;
    const float* st = slot + ln.rows * 64 + (16 * j + c) * 2;
    const float mi = st[0], li = st[1];
    const float mn = fmaxf(m, mi), ms = mn == -INFINITY ? 0.f : mn;
    const float fa = __builtin_amdgcn_exp2f(m - ms), fb = __builtin_amdgcn_exp2f(mi - ms);
    m = mn;
    l = l * fa + li * fb;
#pragma unroll
    for (int nb = 0; nb < 4; ++nb)
      x[nb] = x[nb] * fa + *reinterpret_cast<const ba_v4f*>(sums + 16 * nb + 4 * g) * fb;
  }
  // into fp16's range by a power of two of the row
  float xm = 0.f;
  const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
  for (int nb = 0; nb < 4; ++nb) {
    x[nb] *= inv;
#pragma unroll
    for (int r = 0; r < 4; ++r) xm = fmaxf(xm, fabsf(x[nb][r]));
  }
  xm = fmaxf(xm, __shfl_xor(xm, 16, 64));
  xm = fmaxf(xm, __shfl_xor(xm, 32, 64));
  const int e = ba_exponent(xm);
#pragma unroll
  for (int nb = 0; nb < 4; ++nb) x[nb] *= ldexpf(1.f, 4 - e);
  ba_rotate_back<PREC>(a.vrot16, x, lane, out);
  if (row >= it.nrows) return;
  const int ti = row / a.G, tok = it.tok0 + ti, qh = h * a.G + (row - ti * a.G);
#pragma unroll
  for (int ob = 0; ob < 4; ++ob) ba_store(a, tok, qh, 16 * ob + 4 * g, out[ob] * ldexpf(1.f, e - 4));
  if (a.lse && g == 0) a.lse[(int64_t)tok * a.hq + qh] = ba_lse(m, l);
}

// --------------------------------------------------------------------------------- plans

// Which kernels a call runs, and its workspace.
struct BaPlan {
  bool prec, pair;
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
  TQ_REQUIRE(n_seqs < kBaMaxSegs && n_groups <= kBaMaxSegs, "a call takes at most %d sequences and %d groups, got %d and %d",
             kBaMaxSegs - 1, kBaMaxSegs, n_seqs, n_groups);
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
  TQ_REQUIRE(v.softcap >= 0.f && v.softcap < INFINITY, "softcap must be finite and not negative, got %g", v.softcap);
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
  a.direct = n_groups == 0 && p.groups[0] > 1;
  // waves of several rounds share R_k's parts: about two workgroups a CU at the most
  const int64_t rot = std::min<int64_t>((qrows + 16 * kPrepWaves - 1) / (16 * kPrepWaves), 2 * device_cu_count());
  const dim3 prep((unsigned)(lines + 1 + rot)), pthreads(kPrepThreads);
  if (q_dtype == TQ_F32) hipLaunchKernelGGL((batch_prep_kernel<TQ_F32>), prep, pthreads, 0, st, a, lines, vbits);
  else if (q_dtype == TQ_F16) hipLaunchKernelGGL((batch_prep_kernel<TQ_F16>), prep, pthreads, 0, st, a, lines, vbits);
  else hipLaunchKernelGGL((batch_prep_kernel<TQ_BF16>), prep, pthreads, 0, st, a, lines, vbits);
  TQ_LAUNCH_CHECK("batch_prep_kernel");
  ba_run(vbits, a, p, st);
  TQ_LAUNCH_CHECK("batch_attn_kernel");
  if (a.direct) {
    const dim3 cut((unsigned)((a.line[0].waves - 1) * p.groups[0] + kTailBlocks));
    if (p.prec) hipLaunchKernelGGL((batch_join_cut_kernel<true>), cut, dim3(64), 0, st, a);
    else hipLaunchKernelGGL((batch_join_cut_kernel<false>), cut, dim3(64), 0, st, a);
  } else {
    hipLaunchKernelGGL(batch_join_kernel, dim3((unsigned)((qrows + 15) / 16)), dim3(64 * kJoinWaves), 0, st, a);
  }
  TQ_LAUNCH_CHECK("batch_join_kernel");
  return TQ_OK;
}

}  // extern "C"
