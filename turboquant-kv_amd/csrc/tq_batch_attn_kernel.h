// tq_batch_attn_kernel.h -- the kernel described in tq_batch_attn.h, and ba_launch<VB>.
#pragma once

#include "tq_batch_attn.h"

namespace tq {
namespace {

// LDS: key table, value table, then the scratch area.
constexpr int kBaVTab = 65536;
constexpr int kBaScratch = 131072;
constexpr int kBaNorms = kBaScratch;                       // [8 waves][2][64] floats
constexpr int kBaStats = kBaNorms + kBaWaves * 512;        // [8 waves][48][2] floats
constexpr int kBaMerge = kBaStats + kBaWaves * 48 * 8;     // [8 waves][16][36] floats; rotated queries [48][68]
constexpr int kBaFinal = kBaMerge + kBaWaves * 16 * 36 * 4;  // [16][68] floats
constexpr int kBaSched = kBaFinal + 16 * 68 * 4;
constexpr int kBaLds = kBaSched + 512;
static_assert(kBaLds <= 163840 && 48 * 68 * 4 <= kBaFinal - kBaMerge, "LDS");

__device__ __forceinline__ ba_v8h ba_h8(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  ba_u32x4 t = {a, b, c, d};
  return __builtin_bit_cast(ba_v8h, t);
}

__device__ __forceinline__ uint32_t ba_pack(_Float16 lo, _Float16 hi) {
  typedef _Float16 h2_t __attribute__((ext_vector_type(2)));
  return __builtin_bit_cast(uint32_t, (h2_t){lo, hi});
}

// 2^-e with amax = m 2^e, m in [0.5, 1) (1 for 0, inf or NaN)
__device__ __forceinline__ float ba_pow2_scale(float amax) {
  int e = 0;
  if (amax > 0.f && amax < INFINITY) frexpf(amax, &e);
  return ldexpf(1.f, -e);
}

// cap2 tanh(y / cap2).  tanh z = 1 - 2 / (1 + e^(2 z)), exact at both ends (the exponential
// overflows to inf or vanishes); its absolute error of about 2^-23 is cap2 2^-23 in the score.
// EXACT: below |z| = 0.3 the odd series instead (the next term is 6e-10 relative), whose error
// is relative.
template <bool EXACT>
__device__ __forceinline__ float ba_softcap(float y, float cap2, float cap2_inv) {
  const float z = y * cap2_inv;
  const float e = __builtin_amdgcn_exp2f(z * 2.885390081777927f);
  const float big = fmaf(-2.f * cap2, __builtin_amdgcn_rcpf(1.f + e), cap2);
  if constexpr (!EXACT) {
    return big;
  } else {
    const float w = z * z;
    float p = fmaf(w, -0.00886323552990f, 0.0218694885361f);
    p = fmaf(w, p, -0.0539682539683f);
    p = fmaf(w, p, 0.133333333333f);
    p = fmaf(w, p, -0.333333333333f);
    const float small = fmaf(y * w, p, y);
    return w < 0.09f ? small : big;
  }
}

__device__ __forceinline__ int ba_wave_min(int v) {
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) v = min(v, __shfl_xor(v, o, 64));
  return __builtin_amdgcn_readfirstlane(v);
}
__device__ __forceinline__ int ba_wave_max(int v) { return -ba_wave_min(-v); }

template <int VB, bool SUB, bool PREC, int NGR, bool ROWS>
__global__ __launch_bounds__(kBaThreads, 2) void batch_attn_kernel(BaArgs a) {
#pragma clang fp contract(off)
  constexpr int R = 16 * NGR;                      // rows of a wave
  constexpr int IR = ROWS ? R * kBaWaves : R;      // rows of an item
  __shared__ __attribute__((aligned(16))) uint8_t smem[kBaLds];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int c = lane & 15, g = lane >> 4;
  const int hkv = a.hkv, G = a.G;

  // ---- schedule: this workgroup's piece of the line.  Every thread sums a run of segments.
  const int nseg = a.over_groups ? a.n_groups : a.B + 1;
  int64_t pos, end, chunk, total;
  BaPlace at;
  {
    int64_t* wsum = reinterpret_cast<int64_t*>(smem + kBaSched);        // [8] tiles
    int* wcnt = reinterpret_cast<int*>(smem + kBaSched + 64);           // [8] items
    BaPlace* found = reinterpret_cast<BaPlace*>(smem + kBaSched + 128);
    const int per = (nseg + kBaThreads - 1) / kBaThreads;
    const int s0 = min(nseg, tid * per), s1 = min(nseg, s0 + per);
    int64_t sum = 0;
    int cnt = 0;
    for (int s = s0; s < s1; ++s) {
      const BaSeg x = ba_segment(a, s, IR);
      cnt += x.nrt;
      if constexpr (ROWS) {
        sum += (int64_t)x.nrt * hkv;
      } else {
        for (int rt = 0; rt < x.nrt; ++rt) {
          int t0, nt;
          ba_range(a, x, rt, IR, t0, nt);
          sum += (int64_t)max(1, nt) * hkv;
        }
      }
    }
    int64_t isum = sum;
    int icnt = cnt;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int64_t us = __shfl_up(isum, o, 64);
      const int uc = __shfl_up(icnt, o, 64);
      if (lane >= o) {
        isum += us;
        icnt += uc;
      }
    }
    if (lane == 63) {
      wsum[wave] = isum;
      wcnt[wave] = icnt;
    }
    __syncthreads();
    int64_t bs = 0;
    int bc = 0, items = 0;
    total = 0;
#pragma unroll
    for (int w = 0; w < kBaWaves; ++w) {
      if (w < wave) {
        bs += wsum[w];
        bc += wcnt[w];
      }
      total += wsum[w];
      items += wcnt[w];
    }
    bs += isum - sum;
    bc += icnt - cnt;
    const int64_t grid = gridDim.x;
    if constexpr (ROWS) {
      chunk = 1;
      pos = total - 1 - (int64_t)blockIdx.x;  // the last rows of a sequence see the most: first
      if (pos < 0) return;
      end = pos + 1;
    } else {
      // a piece is eight tiles at least: one per wave
      chunk = max<int64_t>(kBaWaves, (total + grid - 1) / grid);
      // neighbours on the line on one XCD (workgroup w runs on XCD w % 8): adjacent KV heads
      // of a 16-token block share cache lines of norms
      const int64_t w = grid % 8 == 0 ? (blockIdx.x % 8) * (grid / 8) + blockIdx.x / 8 : blockIdx.x;
      pos = w * chunk;
      end = min(pos + chunk, total);
      if (w == 0 && tid == 0) {
        a.head->chunk = chunk;
        a.head->n_items = items;
      }
      if (pos >= total) return;
    }
    if (sum > 0 && pos >= bs && pos < bs + sum) {
      int64_t rel = pos - bs;
      int item = bc;
      for (int s = s0; s < s1; ++s) {
        const BaSeg x = ba_segment(a, s, IR);
        bool here = false;
        int rt = 0;
        if constexpr (ROWS) {
          if (rel < (int64_t)x.nrt * hkv) {
            rt = (int)(rel / hkv);
            rel -= (int64_t)rt * hkv;
            item += rt;
            here = true;
          } else {
            rel -= (int64_t)x.nrt * hkv;
            item += x.nrt;
          }
        } else {
          for (; rt < x.nrt; ++rt) {
            int t0, nt;
            ba_range(a, x, rt, IR, t0, nt);
            const int64_t span = (int64_t)max(1, nt) * hkv;
            if (rel < span) {
              here = true;
              break;
            }
            rel -= span;
            ++item;
          }
        }
        if (here) {
          *found = BaPlace{s, rt, item, rel};
          break;
        }
      }
    }
    __syncthreads();
    at = *found;
    at.seg = __builtin_amdgcn_readfirstlane(at.seg);
    at.rt = __builtin_amdgcn_readfirstlane(at.rt);
    at.item = __builtin_amdgcn_readfirstlane(at.item);
    at.at = (int64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)at.at) |
            (int64_t)__builtin_amdgcn_readfirstlane((int)(at.at >> 32)) << 32;
  }

  // ---- centroid tables scaled by powers of two into [0.5, 1): fp16 hi (and lo) parts
  float ksc, vsc;
  {
    float* sc = reinterpret_cast<float*>(smem + kBaMerge);
    if (wave == 0) {
      const float km = wave_max(lane < 16 ? fabsf(a.kcen[lane]) : 0.f);
      const float vm = wave_max(lane < (1 << VB) ? fabsf(a.vcen[lane]) : 0.f);
      if (lane == 0) {
        sc[0] = ba_pow2_scale(km);
        sc[1] = ba_pow2_scale(vm);
      }
    }
    __syncthreads();
    ksc = sc[0];
    vsc = sc[1];
    const int e = tid & 255, half = tid >> 8;  // threads t and t + 256 write half an entry's copies each
    ba_u32x4 kq, vq[1];
    {
      const float c0 = a.kcen[e >> 4] * ksc, c1 = a.kcen[e & 15] * ksc;
      const _Float16 h0 = (_Float16)c0, h1 = (_Float16)c1;
      const uint32_t hi = ba_pack(h0, h1);
      const uint32_t lo = ba_pack((_Float16)(c0 - (float)h0), (_Float16)(c1 - (float)h1));
      kq = PREC ? (ba_u32x4){hi, lo, hi, lo} : (ba_u32x4){hi, hi, hi, hi};
    }
    if constexpr (VB == 2) {  // the centroids of a byte's four tokens
      _Float16 vh[4], vl[4];
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        const float v = a.vcen[(e >> (2 * t)) & 3] * vsc;
        vh[t] = (_Float16)v;
        vl[t] = (_Float16)(v - (float)vh[t]);
      }
      const uint32_t h0 = ba_pack(vh[0], vh[1]), h1 = ba_pack(vh[2], vh[3]);
      vq[0] = PREC ? (ba_u32x4){h0, h1, ba_pack(vl[0], vl[1]), ba_pack(vl[2], vl[3])}
                   : (ba_u32x4){h0, h1, h0, h1};
    } else {  // of a token pair (3 bits: the byte's top two bits belong to another dim)
      constexpr int mask = (1 << VB) - 1;
      const float x0 = a.vcen[e & mask] * vsc, x1 = a.vcen[(e >> VB) & mask] * vsc;
      const _Float16 y0 = (_Float16)x0, y1 = (_Float16)x1;
      const uint32_t hi = ba_pack(y0, y1);
      const uint32_t lo = ba_pack((_Float16)(x0 - (float)y0), (_Float16)(x1 - (float)y1));
      vq[0] = PREC ? (ba_u32x4){hi, lo, hi, lo} : (ba_u32x4){hi, hi, hi, hi};
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      // rotated by the entry so that a wave's stores spread over the banks
      const int o = e * 256 + half * 128 + 16 * ((j + e) & 7);
      *reinterpret_cast<ba_u32x4*>(smem + o) = kq;
      *reinterpret_cast<ba_u32x4*>(smem + kBaVTab + o) = vq[0];
    }
    __syncthreads();
  }
  // this lane's copy of an entry, and (byte 1) the value table's base
  const uint32_t koff = PREC ? 8u * (lane & 31) : 4u * lane;
  const uint32_t voff = (VB == 2 ? (PREC ? 16u * (lane & 15) : 8u * (lane & 31)) : (PREC ? 8u * (lane & 31) : 4u * lane));
  // address of byte i of w: entry i * 256 + copy
  auto kaddr = [&](uint32_t w, int i) -> uint32_t {
    return __builtin_amdgcn_perm(koff, w, 0x0c0c0004u | ((uint32_t)i << 8));
  };
  auto vaddr = [&](uint32_t w, int i) -> uint32_t {
    return __builtin_amdgcn_perm(voff, w, 0x0c0c0004u | ((uint32_t)i << 8));
  };

  const int bsl = a.bs_log2;
  float* const snorm = reinterpret_cast<float*>(smem + kBaNorms) + wave * 128;
  const bool mods = a.cap2 != 0.f || a.slopes != nullptr;

  for (;;) {  // pieces
    const BaSeg sg = ba_segment(a, at.seg, IR);
    int t0, nt;
    ba_range(a, sg, at.rt, IR, t0, nt);
    const int cost = ROWS ? 1 : max(1, nt);
    const int h = (int)(at.at / cost);
    const int off = (int)(at.at - (int64_t)h * cost);  // tiles of this (item, head) before the piece
    const int n = ROWS ? 1 : (int)min<int64_t>(cost - off, end - pos);
    const int nrows = sg.ntok * G;
    const int irow = at.rt * IR + (ROWS ? wave * R : 0);
    if (!ROWS && off == 0 && h == 0 && tid == 0) {
      // (starts that do not ascend could make more items than there is room for)
      if (at.item < a.max_items) a.items[at.item] = BaItem{pos, cost, at.seg, at.rt, 0};
      if (a.over_groups && at.rt == 0) a.seg_item[at.seg] = at.item;
    }
    const int lastrow = nrows - 1;

    if (!ROWS || irow < nrows) {
      // ---- rows: group j of the wave holds rows irow + 16 j + c (past the end: the last)
      int tok[NGR], qh[NGR], lo[NGR], hi[NGR], qpos[NGR];
      float slope[NGR];
#pragma unroll
      for (int j = 0; j < NGR; ++j) {
        const int row = min(irow + 16 * j + c, lastrow);
        const int ti = row / G;
        tok[j] = sg.tok0 + ti;
        qh[j] = h * G + (row - ti * G);
        int p = sg.past + ti, pl = sg.prefix, top = sg.hi;
        if (a.over_groups) {
          const int b = sg.b0 + ba_last(sg.b1 - sg.b0, tok[j], [&](int i) { return ba_qs(a, sg.b0 + i); });
          const int q0 = ba_qs(a, b), T = max(0, a.seq_lens[b]);
          p = T - (ba_qs(a, b + 1) - q0) + (tok[j] - q0);
          pl = a.prefix_lens ? a.prefix_lens[b] : 0;
          top = min(top, T);
        }
        qpos[j] = p;
        hi[j] = (int)min<int64_t>(top, max<int64_t>((int64_t)p + 1, pl));
        int64_t l64 = sg.lo;
        if (a.window > 0) l64 = max<int64_t>(l64, (int64_t)p + 1 - a.window);
        if (a.token_starts && sg.hi > 0) l64 = max<int64_t>(l64, a.token_starts[tok[j]]);
        lo[j] = (int)min<int64_t>(l64, INT_MAX);
        slope[j] = a.slopes ? a.slopes[qh[j]] * 1.4426950408889634f : 0.f;
      }
      int lo_min = INT_MAX, lo_max = 0, hi_min = INT_MAX, hi_max = 0;
#pragma unroll
      for (int j = 0; j < NGR; ++j) {
        lo_min = min(lo_min, lo[j]);
        lo_max = max(lo_max, lo[j]);
        hi_min = min(hi_min, hi[j]);
        hi_max = max(hi_max, hi[j]);
      }
      lo_min = ba_wave_min(lo_min);
      lo_max = ba_wave_max(lo_max);
      hi_min = ba_wave_min(hi_min);
      hi_max = ba_wave_max(hi_max);
      // tiles that some row of the wave sees, of the piece's
      int k0 = t0 + (ROWS ? 0 : off), k1 = ROWS ? t0 + nt : min(t0 + nt, k0 + n);
      const int skip = max(k0, lo_min >> 6);
      constexpr int kStep = ROWS ? 1 : kBaWaves;
      k0 = ROWS ? skip : skip + wave;
      k1 = hi_max > lo_min ? min(k1, (int)(((int64_t)hi_max + 63) >> 6)) : k0;
      const int nw = k1 > k0 ? (k1 - k0 + kStep - 1) / kStep : 0;

      // ---- Qrot = (q * qscale) R_k^T.  MFMA mb, k-step s: lane (c, g) supplies A[c][g] =
      // R_k[16 (c / 4) + 4 mb + c % 4][16 g + s] and B[g][c] = q_c[16 g + s]; register r of lane
      // (c, g) gets Qrot_c[16 g + 4 mb + r]: a lane ends with dims 16 g .. 16 g + 15, the order
      // in which its key bytes come.
      ba_v8h qhi[NGR][2], qlo[PREC ? NGR : 1][2];
      float kinv[NGR];
      auto load_q = [&](int j, float* qv) {
        const int64_t qo = (int64_t)tok[j] * a.q_stride + qh[j] * 64 + 16 * g;
        if (a.q_dt == TQ_F32) {
          const ba_v4f* src = reinterpret_cast<const ba_v4f*>(static_cast<const float*>(a.q) + qo);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const ba_v4f v = src[i];
            qv[4 * i] = v.x; qv[4 * i + 1] = v.y; qv[4 * i + 2] = v.z; qv[4 * i + 3] = v.w;
          }
        } else {
          const ba_u32x4* src = reinterpret_cast<const ba_u32x4*>(static_cast<const uint16_t*>(a.q) + qo);
          const bool bf = a.q_dt == TQ_BF16;
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const ba_u32x4 v = src[i];
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              const uint32_t hb = (v[e >> 1] >> (16 * (e & 1))) & 0xFFFFu;
              qv[8 * i + e] = bf ? __uint_as_float(hb << 16) : (float)__builtin_bit_cast(_Float16, (uint16_t)hb);
            }
          }
        }
      };
      auto load_rk = [&](int mb, float* rk) {
        const ba_v4f* src = reinterpret_cast<const ba_v4f*>(a.krot + (16 * (c >> 2) + 4 * mb + (c & 3)) * 64 + 16 * g);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const ba_v4f v = src[i];
          rk[4 * i] = v.x; rk[4 * i + 1] = v.y; rk[4 * i + 2] = v.z; rk[4 * i + 3] = v.w;
        }
      };
      auto rotate = [&](const float* rk, const float* qv) {
        ba_v4f d = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int s = 0; s < 16; ++s) d = __builtin_amdgcn_mfma_f32_16x16x4f32(rk[s], qv[s] * a.qscale, d, 0, 0, 0);
        return d;
      };
      auto take_q = [&](int j, const ba_v4f* d) {  // hi + lo parts of a row's 16 dims, scaled by a power of two
        float qm = 0.f;
#pragma unroll
        for (int mb = 0; mb < 4; ++mb)
#pragma unroll
          for (int r = 0; r < 4; ++r) qm = fmaxf(qm, fabsf(d[mb][r]));
        qm = fmaxf(qm, __shfl_xor(qm, 16, 64));
        qm = fmaxf(qm, __shfl_xor(qm, 32, 64));
        const float qsc = ba_pow2_scale(qm);
        kinv[j] = 1.f / (qsc * ksc);  // a power of two
#pragma unroll
        for (int s = 0; s < 2; ++s)
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const float v = d[2 * s + (i >> 2)][i & 3] * qsc;
            const _Float16 hv = (_Float16)v;
            qhi[j][s][i] = hv;
            if constexpr (PREC) qlo[j][s][i] = (_Float16)(v - (float)hv);
          }
      };
      if constexpr (ROWS) {
        ba_v4f d[NGR][4];
        float qv[NGR][16];
#pragma unroll
        for (int j = 0; j < NGR; ++j) load_q(j, qv[j]);
#pragma unroll
        for (int mb = 0; mb < 4; ++mb) {
          float rk[16];
          load_rk(mb, rk);
#pragma unroll
          for (int j = 0; j < NGR; ++j) d[j][mb] = rotate(rk, qv[j]);
        }
#pragma unroll
        for (int j = 0; j < NGR; ++j) take_q(j, d[j]);
      } else {
        // the waves share the products: part u = (group, mb)
        float* qrot = reinterpret_cast<float*>(smem + kBaMerge);  // [R][68]
        for (int u = wave; u < 4 * NGR; u += kBaWaves) {
          float rk[16], qv[16];
          load_rk(u & 3, rk);
#pragma unroll
          for (int j = 0; j < NGR; ++j)
            if (j == (u >> 2)) load_q(j, qv);
          const ba_v4f d = rotate(rk, qv);
          *reinterpret_cast<ba_v4f*>(qrot + (16 * (u >> 2) + c) * 68 + 16 * g + 4 * (u & 3)) = d;
        }
        __syncthreads();
#pragma unroll
        for (int j = 0; j < NGR; ++j) {
          ba_v4f d[4];
#pragma unroll
          for (int mb = 0; mb < 4; ++mb)
            d[mb] = *reinterpret_cast<const ba_v4f*>(qrot + (16 * j + c) * 68 + 16 * g + 4 * mb);
          take_q(j, d);
        }
      }

      // ---- tiles
      float m[NGR], l[NGR];
      ba_v4f o[NGR][4];
      VnScale vs;
#pragma unroll
      for (int j = 0; j < NGR; ++j) {
        m[j] = -INFINITY;
        l[j] = 0.f;
#pragma unroll
        for (int nb = 0; nb < 4; ++nb) o[j][nb] = (ba_v4f){0.f, 0.f, 0.f, 0.f};
      }

      // Block ids of 16 tiles at a time, the next 16 requested while these are used: lane
      // 4 i + b holds the block of tile i's 16-token group b.
      const int32_t* btab = a.block_tables + (int64_t)sg.table * a.table_stride;
      auto load_ids = [&](int chunk16) -> uint32_t {
        const int i = min(chunk16 * 16 + (lane >> 2), nw - 1);
        const int64_t tb = ((int64_t)(k0 + (int64_t)i * kStep) << 6) + 16 * (lane & 3);
        const int bi = (int)min<int64_t>(tb >> bsl, (int64_t)a.max_blocks - 1);
        return min((uint32_t)btab[bi], a.num_blocks - 1u);
      };
      constexpr int NV = VB == 2 ? 4 : (SUB ? 8 : 2 * VB);
      struct Tile {
        ba_u32x2 kw[4];
        float nk, nv;
        uint32_t vw[NV];
      };
      uint32_t ids = 0, ids_next = 0;
      if (nw > 0) {
        ids_next = load_ids(0);
      }
      // i: the wave's i-th tile, asked for in order (a repeated last one excepted)
      auto load = [&](int i, Tile& t) {
        if ((i & 15) == 0 && i < nw) {
          ids = ids_next;
          ids_next = load_ids((i >> 4) + 1);
        }
        const int il = min(i, nw - 1);
        const int64_t tb0 = (int64_t)(k0 + (int64_t)il * kStep) << 6;
        const int64_t bsm = ((int64_t)1 << bsl) - 1;
        int64_t base[4];
#pragma unroll
        for (int b = 0; b < 4; ++b) {
          if (SUB || b == 0) {
            const uint32_t blk = (uint32_t)__builtin_amdgcn_readlane((int)ids, 4 * (il & 15) + b);
            base[b] = (((int64_t)blk * hkv + h) << bsl) + ((tb0 + 16 * b) & bsm);
          } else {
            base[b] = base[0] + 16 * b;
          }
        }
#pragma unroll
        for (int b = 0; b < 4; ++b)
          t.kw[b] = *reinterpret_cast<const ba_u32x2*>(a.kpairs + base[b] * 32 + (c * 32 + 8 * g));
        {
          const int64_t nbase = SUB ? (g == 0 ? base[0] : g == 1 ? base[1] : g == 2 ? base[2] : base[3]) + c
                                    : base[0] + lane;
          t.nk = a.knorms[nbase];
          t.nv = a.vnorms[nbase];
        }
        if constexpr (SUB) {
#pragma unroll
          for (int b = 0; b < 4; ++b) {
            const uint8_t* sb = a.vtiles + base[b] * (8 * VB);
            if constexpr (VB == 2) {
              t.vw[b] = *reinterpret_cast<const uint32_t*>(sb + 4 * lane);
            } else if constexpr (VB == 4) {
              const ba_u32x2 w = *reinterpret_cast<const ba_u32x2*>(sb + 8 * lane);
              t.vw[2 * b] = w.x;
              t.vw[2 * b + 1] = w.y;
            } else {
              t.vw[b] = *reinterpret_cast<const uint32_t*>(sb + 4 * lane);
              t.vw[4 + b] = *reinterpret_cast<const uint16_t*>(sb + 256 + 2 * lane);
            }
          }
        } else {
          const uint8_t* tb = a.vtiles + base[0] * (8 * VB);
          const ba_u32x4 v = *reinterpret_cast<const ba_u32x4*>(tb + 16 * lane);
          t.vw[0] = v.x; t.vw[1] = v.y; t.vw[2] = v.z; t.vw[3] = v.w;
          if constexpr (VB == 3) {
            const ba_u32x2 v1 = *reinterpret_cast<const ba_u32x2*>(tb + 1024 + 8 * lane);
            t.vw[4] = v1.x; t.vw[5] = v1.y;
          } else if constexpr (VB == 4) {
            const ba_u32x4 v1 = *reinterpret_cast<const ba_u32x4*>(tb + 1024 + 16 * lane);
            t.vw[4] = v1.x; t.vw[5] = v1.y; t.vw[6] = v1.z; t.vw[7] = v1.w;
          }
        }
      };

      auto compute = [&](int i, const Tile& t) {
        const int p0 = (k0 + i * kStep) << 6;  // position of the tile's first token
        // norms of tokens no row of the wave sees may be stale, even NaN
        const bool live = p0 + lane >= lo_min && p0 + lane < hi_max;
        const float nvl = live ? t.nv : 0.f;
        if (vs.over(fabsf(nvl) * vs.s)) {
          const float f = vs.rescale(fabsf(nvl));
#pragma unroll
          for (int j = 0; j < NGR; ++j)
#pragma unroll
            for (int nb = 0; nb < 4; ++nb) o[j][nb] *= f;
        }
        snorm[lane] = t.nk;
        snorm[64 + lane] = nvl * vs.s;
        __builtin_amdgcn_wave_barrier();
        const bool mask = p0 < lo_max || p0 + 64 > hi_min;

        // value word helpers: VB 3 / 4, tile word i of half s, and the word whose bytes index
        // the pair entries of dim group nb
        auto tword = [&](int s, int i2) -> uint32_t {
          if constexpr (!SUB) {
            return t.vw[(VB == 4 ? 4 : 3) * s + i2];
          } else if constexpr (VB == 4) {
            return __builtin_amdgcn_perm(t.vw[2 * (2 * s + 1) + (i2 >> 1)], t.vw[2 * (2 * s) + (i2 >> 1)],
                                         (i2 & 1) ? 0x07060302u : 0x05040100u);
          } else {
            return i2 == 2 ? __builtin_amdgcn_perm(t.vw[4 + 2 * s + 1], t.vw[4 + 2 * s], 0x05040100u)
                           : __builtin_amdgcn_perm(t.vw[2 * s + 1], t.vw[2 * s], i2 ? 0x07060302u : 0x05040100u);
          }
        };
        auto vword = [&](int s, int nb) -> uint32_t {
          if constexpr (VB == 4) {
            return tword(s, nb);
          } else {
            if (nb < 3) return tword(s, nb);
            const uint32_t x0 = tword(s, 0), x1 = tword(s, 1), x2 = tword(s, 2);
            return ((x0 >> 6) & 0x03030303u) | ((x1 >> 4) & 0x0C0C0C0Cu) | ((x2 >> 2) & 0x30303030u);
          }
        };

        // ---- scores over the norm's and the scales' powers of two
        ba_v4f sv[NGR][4];
#pragma unroll
        for (int b = 0; b < 4; ++b) {
          ba_v4f acc[NGR];
#pragma unroll
          for (int j = 0; j < NGR; ++j) acc[j] = (ba_v4f){0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int s = 0; s < 2; ++s) {
            const uint32_t w = t.kw[b][s];
            ba_v8h ah, al;
            if constexpr (PREC) {
              const ba_u32x2 e0 = *reinterpret_cast<const ba_u32x2*>(smem + kaddr(w, 0));
              const ba_u32x2 e1 = *reinterpret_cast<const ba_u32x2*>(smem + kaddr(w, 1));
              const ba_u32x2 e2 = *reinterpret_cast<const ba_u32x2*>(smem + kaddr(w, 2));
              const ba_u32x2 e3 = *reinterpret_cast<const ba_u32x2*>(smem + kaddr(w, 3));
              ah = ba_h8(e0.x, e1.x, e2.x, e3.x);
              al = ba_h8(e0.y, e1.y, e2.y, e3.y);
            } else {
              ah = ba_h8(*reinterpret_cast<const uint32_t*>(smem + kaddr(w, 0)),
                         *reinterpret_cast<const uint32_t*>(smem + kaddr(w, 1)),
                         *reinterpret_cast<const uint32_t*>(smem + kaddr(w, 2)),
                         *reinterpret_cast<const uint32_t*>(smem + kaddr(w, 3)));
            }
#pragma unroll
            for (int j = 0; j < NGR; ++j) {
              acc[j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ah, qhi[j][s], acc[j], 0, 0, 0);
              if constexpr (PREC) {
                acc[j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ah, qlo[j][s], acc[j], 0, 0, 0);
                acc[j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(al, qhi[j][s], acc[j], 0, 0, 0);
              }
            }
          }
          const ba_v4f nk4 = *reinterpret_cast<const ba_v4f*>(snorm + 16 * b + 4 * g);
#pragma unroll
          for (int j = 0; j < NGR; ++j)
#pragma unroll
            for (int r = 0; r < 4; ++r) sv[j][b][r] = acc[j][r] * nk4[r];
        }
        if (mods) {  // to the log2 domain, capped and biased
#pragma unroll
          for (int j = 0; j < NGR; ++j) {
            const float d0 = (float)(p0 + 4 * g - qpos[j]);
#pragma unroll
            for (int b = 0; b < 4; ++b)
#pragma unroll
              for (int r = 0; r < 4; ++r) {
                float y = sv[j][b][r] * kinv[j];
                if (a.cap2 != 0.f) y = ba_softcap<PREC>(y, a.cap2, a.cap2_inv);
                sv[j][b][r] = fmaf(slope[j], d0 + (float)(16 * b + r), y);
              }
          }
        }
        if (mask) {
#pragma unroll
          for (int j = 0; j < NGR; ++j) {
            const int rlo = lo[j] - p0 - 4 * g, rhi = hi[j] - p0 - 4 * g;
#pragma unroll
            for (int b = 0; b < 4; ++b)
#pragma unroll
              for (int r = 0; r < 4; ++r)
                sv[j][b][r] = 16 * b + r >= rlo && 16 * b + r < rhi ? sv[j][b][r] : -INFINITY;
          }
        }

        // ---- online softmax (log2 domain); weights times value norms as fp16
        ba_v4f nv4[4];
#pragma unroll
        for (int b = 0; b < 4; ++b) nv4[b] = *reinterpret_cast<const ba_v4f*>(snorm + 64 + 16 * b + 4 * g);
        ba_v8h bh[NGR][2], bl[PREC ? NGR : 1][2];
#pragma unroll
        for (int j = 0; j < NGR; ++j) {
          float mx = -INFINITY;
#pragma unroll
          for (int b = 0; b < 4; ++b)
#pragma unroll
            for (int r = 0; r < 4; ++r) mx = fmaxf(mx, sv[j][b][r]);
          mx = fmaxf(mx, __shfl_xor(mx, 16, 64));
          mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
          const float kin = mods ? 1.f : kinv[j];
          const float mn = fmaxf(m[j], mx * kin);
          const float ms = mn == -INFINITY ? 0.f : mn;
          if (__any(mn != m[j])) {
            const float alpha = __builtin_amdgcn_exp2f(m[j] - ms);
            l[j] *= alpha;
#pragma unroll
            for (int nb = 0; nb < 4; ++nb) o[j][nb] *= alpha;
          }
          m[j] = mn;
          float v[4][4];
#pragma unroll
          for (int b = 0; b < 4; ++b)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
              // results below 2^-126 flush to 0: nothing beside the running maximum's 1
              const float p = __builtin_amdgcn_exp2f(fmaf(sv[j][b][r], kin, -ms));
              l[j] += p;
              v[b][r] = p * nv4[b][r];
              if (mask) v[b][r] = p > 0.f ? v[b][r] : 0.f;  // another row's inf or NaN norm
            }
#pragma unroll
          for (int b = 0; b < 4; ++b)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
              if constexpr (PREC) {
                _Float16 hv, lv;
                split_f16(v[b][r], hv, lv);
                bh[j][b >> 1][4 * (b & 1) + r] = hv;
                bl[j][b >> 1][4 * (b & 1) + r] = lv;
              } else {
                bh[j][b >> 1][4 * (b & 1) + r] = (_Float16)v[b][r];
              }
            }
        }
        // wait states between the conversions and the products that read them
        if constexpr (NGR == 3 && !PREC) {
          mfma_operand_fence6(bh[0][0], bh[0][1], bh[1][0], bh[1][1], bh[2][0], bh[2][1]);
        } else if constexpr (NGR == 2 && PREC) {
          mfma_operand_fence8(bh[0][0], bh[0][1], bh[1][0], bh[1][1], bl[0][0], bl[0][1], bl[1][0], bl[1][1]);
        } else {
#pragma unroll
          for (int j = 0; j < NGR; ++j) {
            if constexpr (PREC) mfma_operand_fence(bh[j][0], bh[j][1], bl[j][0], bl[j][1]);
            else mfma_operand_fence(bh[j][0], bh[j][1]);
          }
        }

        // ---- values
#pragma unroll
        for (int s = 0; s < 2; ++s) {
#pragma unroll
          for (int nb = 0; nb < 4; ++nb) {
            ba_v8h ah, al;
            const uint8_t* vt = smem + kBaVTab;
            if constexpr (VB == 2) {
              const uint32_t a0 = vaddr(t.vw[2 * s], nb), a1 = vaddr(t.vw[2 * s + 1], nb);
              if constexpr (PREC) {
                const ba_u32x4 e0 = *reinterpret_cast<const ba_u32x4*>(vt + a0);
                const ba_u32x4 e1 = *reinterpret_cast<const ba_u32x4*>(vt + a1);
                ah = ba_h8(e0.x, e0.y, e1.x, e1.y);
                al = ba_h8(e0.z, e0.w, e1.z, e1.w);
              } else {
                const ba_u32x2 e0 = *reinterpret_cast<const ba_u32x2*>(vt + a0);
                const ba_u32x2 e1 = *reinterpret_cast<const ba_u32x2*>(vt + a1);
                ah = ba_h8(e0.x, e0.y, e1.x, e1.y);
              }
            } else {
              const uint32_t w = vword(s, nb);
              if constexpr (PREC) {
                const ba_u32x2 e0 = *reinterpret_cast<const ba_u32x2*>(vt + vaddr(w, 0));
                const ba_u32x2 e1 = *reinterpret_cast<const ba_u32x2*>(vt + vaddr(w, 1));
                const ba_u32x2 e2 = *reinterpret_cast<const ba_u32x2*>(vt + vaddr(w, 2));
                const ba_u32x2 e3 = *reinterpret_cast<const ba_u32x2*>(vt + vaddr(w, 3));
                ah = ba_h8(e0.x, e1.x, e2.x, e3.x);
                al = ba_h8(e0.y, e1.y, e2.y, e3.y);
              } else {
                ah = ba_h8(*reinterpret_cast<const uint32_t*>(vt + vaddr(w, 0)),
                           *reinterpret_cast<const uint32_t*>(vt + vaddr(w, 1)),
                           *reinterpret_cast<const uint32_t*>(vt + vaddr(w, 2)),
                           *reinterpret_cast<const uint32_t*>(vt + vaddr(w, 3)));
              }
            }
#pragma unroll
            for (int j = 0; j < NGR; ++j) {
              o[j][nb] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ah, bh[j][s], o[j][nb], 0, 0, 0);
              if constexpr (PREC) {
                o[j][nb] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ah, bl[j][s], o[j][nb], 0, 0, 0);
                o[j][nb] = __builtin_amdgcn_mfma_f32_16x16x32_f16(al, bh[j][s], o[j][nb], 0, 0, 0);
              }
            }
          }
        }
      };

      // Three buffers, two tiles ahead; whole groups of three, then the rest.
      if (nw > 0) {
        Tile r0, r1, r2;
        load(0, r0);
        load(1, r1);
        int i = 0;
        for (; i + 2 < nw; i += 3) {
          load(i + 2, r2);
          compute(i, r0);
          load(i + 3, r0);
          compute(i + 1, r1);
          load(i + 4, r1);
          compute(i + 2, r2);
        }
        if (i < nw) compute(i, r0);
        if (i + 1 < nw) compute(i + 1, r1);
      }
      // the row's sum over its four lanes
#pragma unroll
      for (int j = 0; j < NGR; ++j) {
        l[j] += __shfl_xor(l[j], 16, 64);
        l[j] += __shfl_xor(l[j], 32, 64);
      }
      const float vinv = vs.inv() / vsc;  // powers of two
#pragma unroll
      for (int j = 0; j < NGR; ++j)
#pragma unroll
        for (int nb = 0; nb < 4; ++nb) o[j][nb] *= vinv;

      // out_c[16 ob + 4 g + r] of lane (c, g) = sum over k-steps (nb, r) of A[c][g] =
      // R_v[16 nb + 4 g + r][16 ob + c] and B[g][c] = O_c[16 nb + 4 g + r]
      auto load_rv = [&](int ob, float* rv) {
#pragma unroll
        for (int nb = 0; nb < 4; ++nb)
#pragma unroll
          for (int r = 0; r < 4; ++r) rv[4 * nb + r] = a.vrot[(16 * nb + 4 * g + r) * 64 + 16 * ob + c];
      };
      auto store = [&](int j, int ob, ba_v4f acc) {
        const int64_t oa = (int64_t)tok[j] * a.out_stride + qh[j] * 64 + 16 * ob + 4 * g;
        if (a.q_dt == TQ_F32) {
          *reinterpret_cast<ba_v4f*>(static_cast<float*>(a.out) + oa) = acc;
        } else if (a.q_dt == TQ_BF16) {
          typedef __bf16 b4_t __attribute__((ext_vector_type(4)));
          *reinterpret_cast<b4_t*>(static_cast<uint16_t*>(a.out) + oa) = __builtin_convertvector(acc, b4_t);
        } else {
          typedef _Float16 h4_t __attribute__((ext_vector_type(4)));
          *reinterpret_cast<h4_t*>(static_cast<uint16_t*>(a.out) + oa) = __builtin_convertvector(acc, h4_t);
        }
      };
      const bool tail = !a.over_groups && at.seg == a.B;
      const bool writes = !tail || a.zero_tail;

      if constexpr (ROWS) {
#pragma unroll
        for (int ob = 0; ob < 4; ++ob) {
          float rv[16];
          load_rv(ob, rv);
#pragma unroll
          for (int j = 0; j < NGR; ++j) {
            const float inv = l[j] == 0.f ? 0.f : 1.f / l[j];
            ba_v4f acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int nb = 0; nb < 4; ++nb)
#pragma unroll
              for (int r = 0; r < 4; ++r)
                acc = __builtin_amdgcn_mfma_f32_16x16x4f32(rv[4 * nb + r], o[j][nb][r] * inv, acc, 0, 0, 0);
            if (irow + 16 * j + c <= lastrow && writes) store(j, ob, acc);
          }
        }
        if (a.lse && g == 0) {
#pragma unroll
          for (int j = 0; j < NGR; ++j)
            if (irow + 16 * j + c <= lastrow)
              a.lse[(int64_t)tok[j] * a.hq + qh[j]] =
                  l[j] == 0.f ? -INFINITY : (m[j] + __builtin_amdgcn_logf(l[j])) * 0.6931471805599453f;
        }
      } else {
        // ---- merge the waves: statistics, then the sums, 16 rows and 32 dims at a time
        float* stats = reinterpret_cast<float*>(smem + kBaStats);  // [wave][R][2]
        if (g == 0) {
#pragma unroll
          for (int j = 0; j < NGR; ++j) {
            stats[(wave * R + 16 * j + c) * 2] = m[j];
            stats[(wave * R + 16 * j + c) * 2 + 1] = l[j];
          }
        }
        __syncthreads();
        const bool whole = off == 0 && n == cost;
        // a cut item's piece: slot 1 of its workgroup if it begins here, else slot 0
        float* const slot = whole ? nullptr : a.slots + ((pos / chunk) * 2 + (off == 0)) * ba_slot_floats(R);
        float* const merge = reinterpret_cast<float*>(smem + kBaMerge);  // [wave][16][36]
        float* const fin = reinterpret_cast<float*>(smem + kBaFinal);    // [16][68]
#pragma unroll
        for (int j = 0; j < NGR; ++j) {
          float M = -INFINITY, L = 0.f;
#pragma unroll
          for (int w = 0; w < kBaWaves; ++w) M = fmaxf(M, stats[(w * R + 16 * j + c) * 2]);
          const float Ms = M == -INFINITY ? 0.f : M;
#pragma unroll
          for (int w = 0; w < kBaWaves; ++w)
            L += stats[(w * R + 16 * j + c) * 2 + 1] * __builtin_amdgcn_exp2f(stats[(w * R + 16 * j + c) * 2] - Ms);
          const float f = __builtin_amdgcn_exp2f(m[j] - Ms);
#pragma unroll
          for (int hf = 0; hf < 2; ++hf) {
#pragma unroll
            for (int nb = 0; nb < 2; ++nb)
              *reinterpret_cast<ba_v4f*>(merge + (wave * 16 + c) * 36 + 16 * nb + 4 * g) = o[j][2 * hf + nb] * f;
            __syncthreads();
            const int row = tid >> 5, dim = tid & 31;
            float s = 0.f;
#pragma unroll
            for (int w = 0; w < kBaWaves; ++w) s += merge[(w * 16 + row) * 36 + dim];
            fin[row * 68 + 32 * hf + dim] = s;
            __syncthreads();
          }
          if (whole && !a.row_sums) {
            const float inv = L == 0.f ? 0.f : 1.f / L;
            if (wave < 4) {
              float rv[16];
              load_rv(wave, rv);
              ba_v4f acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
              for (int nb = 0; nb < 4; ++nb) {
                const ba_v4f x = *reinterpret_cast<const ba_v4f*>(fin + c * 68 + 16 * nb + 4 * g);
#pragma unroll
                for (int r = 0; r < 4; ++r)
                  acc = __builtin_amdgcn_mfma_f32_16x16x4f32(rv[4 * nb + r], x[r] * inv, acc, 0, 0, 0);
              }
              if (irow + 16 * j + c <= lastrow && writes) store(j, wave, acc);
            } else if (wave == 4 && a.lse && g == 0 && irow + 16 * j + c <= lastrow) {
              a.lse[(int64_t)tok[j] * a.hq + qh[j]] =
                  L == 0.f ? -INFINITY : (M + __builtin_amdgcn_logf(L)) * 0.6931471805599453f;
            }
          } else {
            const int row = tid >> 5, dim = 2 * (tid & 31), at_row = irow + 16 * j + row;
            typedef float v2f __attribute__((ext_vector_type(2)));
            const v2f x = *reinterpret_cast<const v2f*>(fin + row * 68 + dim);
            float *sums, *st;
            if (slot) {
              sums = slot + (16 * j + row) * 64;
              st = slot + R * 64 + (16 * j + c) * 2;
            } else {
              const int ti = min(at_row, lastrow) / G;
              sums = a.row_sums + ((int64_t)(sg.tok0 + ti) * a.hq + h * G + (min(at_row, lastrow) - ti * G)) * 64;
              st = a.row_stats + ((int64_t)tok[j] * a.hq + qh[j]) * 2;
            }
            if (slot || at_row <= lastrow) *reinterpret_cast<v2f*>(sums + dim) = x;
            if (wave == 0 && g == 0 && (slot || irow + 16 * j + c <= lastrow)) {
              st[0] = M;
              st[1] = L;
            }
          }
        }
      }
    }
    if constexpr (ROWS) return;
    pos += n;
    if (pos >= end) return;
    at.at += n;
    if (at.at == (int64_t)cost * hkv) {
      at.at = 0;
      ++at.item;
      if (++at.rt == sg.nrt) {
        at.rt = 0;
        do ++at.seg;
        while (at.seg < nseg && ba_segment(a, at.seg, IR).nrt == 0);
      }
    }
  }
}

}  // namespace

template <int VB, bool SUB, bool PREC>
void ba_launch_kind(const BaArgs& a, bool rows, int groups, unsigned grid, hipStream_t st) {
  constexpr int N = ba_groups(PREC);
  if (rows)
    hipLaunchKernelGGL((batch_attn_kernel<VB, SUB, PREC, N, true>), dim3(grid), dim3(kBaThreads), 0, st, a);
  else if (groups == 1)
    hipLaunchKernelGGL((batch_attn_kernel<VB, SUB, PREC, 1, false>), dim3(grid), dim3(kBaThreads), 0, st, a);
  else
    hipLaunchKernelGGL((batch_attn_kernel<VB, SUB, PREC, N, false>), dim3(grid), dim3(kBaThreads), 0, st, a);
}

template <int VB>
void ba_launch(const BaArgs& a, bool sub, bool prec, bool rows, int groups, unsigned grid, hipStream_t st) {
  if (sub && prec) ba_launch_kind<VB, true, true>(a, rows, groups, grid, st);
  else if (sub) ba_launch_kind<VB, true, false>(a, rows, groups, grid, st);
  else if (prec) ba_launch_kind<VB, false, true>(a, rows, groups, grid, st);
  else ba_launch_kind<VB, false, false>(a, rows, groups, grid, st);
}

}  // namespace tq
