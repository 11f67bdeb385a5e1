// tq_batch_attn_kernel.h -- the main kernel described in tq_batch_attn.h, and ba_launch<VB>.
#pragma once

#include "tq_batch_attn.h"

namespace tq {
namespace {

// LDS: key table, value table, each wave's norms of a tile.
constexpr int kBaVTab = 65536;
constexpr int kBaNorms = 131072;  // [8 waves][2][64] floats
constexpr int kBaLds = kBaNorms + kBaWaves * 512;

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


// The larger of x over the lanes c, c + 16, c + 32, c + 48.
__device__ __forceinline__ float ba_max4(float x) {
  x = fmaxf(x, __shfl_xor(x, 16, 64));
  return fmaxf(x, __shfl_xor(x, 32, 64));
}

// RW rows of 16 columns (16 / RW copies share a tile's tokens), NGR groups of columns.
template <int VB, bool SUB, bool PREC, int RW, int NGR>
__global__ __launch_bounds__(kBaThreads, 2) void batch_attn_kernel(BaArgs a, BaLine ln) {
#pragma clang fp contract(off)
  static_assert(NGR == 1 || RW == 16, "groups of columns hold 16 rows each");
  constexpr int NB = RW / 4;       // 16-token groups whose scores a lane keeps
  constexpr int R = RW * NGR;
  __shared__ __attribute__((aligned(16))) uint8_t smem[kBaLds];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int c = lane & 15, g = lane >> 4;
  const int cb = c / RW, cr = c % RW;  // the column's copy and row
  const int hkv = a.hkv, G = a.G;

  // Neighbouring pieces on one XCD (workgroup w runs on XCD w % 8): rows of one prefix read the
  // same tiles there, and adjacent KV heads of a 16-token block share lines of norms.  Few
  // pieces spread over the workgroups.
  const unsigned grid = gridDim.x;
  const unsigned blk = grid % 8 == 0 ? (blockIdx.x % 8) * (grid / 8) + blockIdx.x / 8 : blockIdx.x;
  if (ln.work[blk] < 0) return;  // the workgroup's first piece: there is none behind the line's end
  const int w = wave * (int)grid + (int)blk;
  int item = ln.work[w];
  const int64_t chunk = ln.head->chunk, total = ln.head->total;

  // ---- centroid tables scaled by powers of two into [0.5, 1): fp16 hi (and lo) parts
  float ksc, vsc;
  {
    float* sc = reinterpret_cast<float*>(smem + kBaNorms);
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
    const int e = tid & 255, half = tid >> 8;  // entry, 128-byte half: the hi parts (PREC: the lo parts in half 1)
    ba_u32x4 kq, vq;
    {
      const float c0 = a.kcen[e >> 4] * ksc, c1 = a.kcen[e & 15] * ksc;
      const _Float16 h0 = (_Float16)c0, h1 = (_Float16)c1;
      const uint32_t hi = ba_pack(h0, h1);
      const uint32_t lo = ba_pack((_Float16)(c0 - (float)h0), (_Float16)(c1 - (float)h1));
      const uint32_t x = PREC && half ? lo : hi;
      kq = (ba_u32x4){x, x, x, x};
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
      const uint32_t l0 = ba_pack(vl[0], vl[1]), l1 = ba_pack(vl[2], vl[3]);
      vq = PREC && half ? (ba_u32x4){l0, l1, l0, l1} : (ba_u32x4){h0, h1, h0, h1};
    } else {  // of a token pair (3 bits: the byte's top two bits belong to another dim)
      constexpr int mask = (1 << VB) - 1;
      const float x0 = a.vcen[e & mask] * vsc, x1 = a.vcen[(e >> VB) & mask] * vsc;
      const _Float16 y0 = (_Float16)x0, y1 = (_Float16)x1;
      const uint32_t hi = ba_pack(y0, y1);
      const uint32_t lo = ba_pack((_Float16)(x0 - (float)y0), (_Float16)(x1 - (float)y1));
      const uint32_t x = PREC && half ? lo : hi;
      vq = (ba_u32x4){x, x, x, x};
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      // rotated by the entry so that a wave's stores spread over the banks
      const int o = e * 256 + half * 128 + 16 * ((j + e) & 7);
      *reinterpret_cast<ba_u32x4*>(smem + o) = kq;
      *reinterpret_cast<ba_u32x4*>(smem + kBaVTab + o) = vq;
    }
    __syncthreads();
  }
  // this lane's copy of an entry's hi part (PREC: its lo part is 128 bytes on)
  const uint32_t koff = PREC ? 4u * (lane & 31) : 4u * lane;
  const uint32_t voff = VB == 2 ? (PREC ? 8u * (lane & 15) : 8u * (lane & 31)) : koff;
  // address of byte i of w: entry i * 256 + copy
  auto kaddr = [&](uint32_t w, int i) -> uint32_t {
    return __builtin_amdgcn_perm(koff, w, 0x0c0c0004u | ((uint32_t)i << 8));
  };
  auto vaddr = [&](uint32_t w, int i) -> uint32_t {
    return __builtin_amdgcn_perm(voff, w, 0x0c0c0004u | ((uint32_t)i << 8));
  };


  if (item < 0) return;
  const int bsl = a.bs_log2;
  float* const snorm = reinterpret_cast<float*>(smem + kBaNorms) + wave * 128;
  const bool mods = a.cap2 != 0.f || a.slopes != nullptr;
  int64_t pos = (int64_t)w * chunk;
  const int64_t end = min(pos + chunk, total);

  while (pos < end) {  // (item, head)s of the piece
    const BaItem it = ln.items[item];
    const int t0 = __builtin_amdgcn_readfirstlane(it.t0), nt = __builtin_amdgcn_readfirstlane(it.nt);
    const int tok0 = __builtin_amdgcn_readfirstlane(it.tok0), row0 = __builtin_amdgcn_readfirstlane(it.row0);
    const int lastrow = __builtin_amdgcn_readfirstlane(it.nrows) - 1;
    const int table = __builtin_amdgcn_readfirstlane(it.table);
    const int cost = nt + kBaOver;
    const int h = __builtin_amdgcn_readfirstlane((int)((pos - it.start) / cost));
    const int off = __builtin_amdgcn_readfirstlane((int)(pos - it.start - (int64_t)h * cost));
    const int n = (int)min<int64_t>(cost - off, end - pos);
    const int ta = (int)ba_tiles(off), tb = (int)ba_tiles(off + n);
    const bool whole = tb - ta == nt && (nt > 0 || off == 0);
    pos += n;
    if (off + n == cost && h == hkv - 1) ++item;
    if (!whole && ta == tb) continue;

    // ---- rows: group j's column c holds row row0 + 16 j + cr (past the end: the last)
    int tok[NGR], qh[NGR], lo[NGR], hi[NGR], qpos[NGR];
    float slope[NGR], kinv[NGR];
    ba_v8h qhi[NGR][2], qlo[PREC ? NGR : 1][2];
#pragma unroll
    for (int j = 0; j < NGR; ++j) {
      const int row = min(row0 + 16 * j + cr, lastrow);
      const int ti = row / G;
      tok[j] = tok0 + ti;
      qh[j] = h * G + (row - ti * G);
      const BaToken t = a.tokens[tok[j]];
      lo[j] = max(t.lo, it.lo);
      hi[j] = min(t.hi, it.hi);
      qpos[j] = t.pos;
      const int64_t rowid = (int64_t)tok[j] * a.hq + qh[j];
      kinv[j] = a.qscale_inv[rowid] / ksc;  // powers of two
      slope[j] = a.slopes ? a.slopes[qh[j]] * 1.4426950408889634f : 0.f;
#pragma unroll
      for (int s = 0; s < 2; ++s) {  // dims 16 g + 8 s ..
        qhi[j][s] = *reinterpret_cast<const ba_v8h*>(a.qhi + rowid * 64 + 16 * g + 8 * s);
        if constexpr (PREC) qlo[j][s] = *reinterpret_cast<const ba_v8h*>(a.qlo + rowid * 64 + 16 * g + 8 * s);
      }
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
    // tiles of the piece that some row sees
    const int k0 = max(t0 + ta, lo_min >> 6);
    const int k1 = hi_max > lo_min ? min(t0 + tb, (int)(((int64_t)hi_max + 63) >> 6)) : k0;
    const int nw = max(0, k1 - k0);

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
    const int32_t* btab = a.block_tables + (int64_t)table * a.table_stride;
    auto load_ids = [&](int chunk16) -> uint32_t {
      const int i = min(chunk16 * 16 + (lane >> 2), nw - 1);
      const int64_t tb = ((int64_t)(k0 + i) << 6) + 16 * (lane & 3);
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
      const int64_t tb0 = (int64_t)(k0 + il) << 6;
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
      const int p0 = (k0 + i) << 6;  // position of the tile's first token
      // norms of tokens no row sees may be stale, even NaN
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


      // ---- scores over the norm's and the scales' powers of two: entry k of a lane is its copy's
      // 16-token group NB cb + k
      ba_v4f sv[NGR][NB];
#pragma unroll
      for (int b = 0; b < 4; ++b) {
        ba_v4f acc[NGR];
#pragma unroll
        for (int j = 0; j < NGR; ++j) acc[j] = (ba_v4f){0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int s = 0; s < 2; ++s) {
          const uint32_t kw = t.kw[b][s];
          const uint8_t* p0a = smem + kaddr(kw, 0);
          const uint8_t* p1a = smem + kaddr(kw, 1);
          const uint8_t* p2a = smem + kaddr(kw, 2);
          const uint8_t* p3a = smem + kaddr(kw, 3);
          const ba_v8h ah = ba_h8(*reinterpret_cast<const uint32_t*>(p0a), *reinterpret_cast<const uint32_t*>(p1a),
                                  *reinterpret_cast<const uint32_t*>(p2a), *reinterpret_cast<const uint32_t*>(p3a));
#pragma unroll
          for (int j = 0; j < NGR; ++j) acc[j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ah, qhi[j][s], acc[j], 0, 0, 0);
          if constexpr (PREC) {
            const ba_v8h al = ba_h8(*reinterpret_cast<const uint32_t*>(p0a + 128), *reinterpret_cast<const uint32_t*>(p1a + 128),
                                    *reinterpret_cast<const uint32_t*>(p2a + 128), *reinterpret_cast<const uint32_t*>(p3a + 128));
#pragma unroll
            for (int j = 0; j < NGR; ++j) {
              acc[j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ah, qlo[j][s], acc[j], 0, 0, 0);
              acc[j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(al, qhi[j][s], acc[j], 0, 0, 0);
            }
          }
        }
#pragma unroll
        for (int j = 0; j < NGR; ++j) {
          if (b / NB == 0) {
            sv[j][b % NB] = acc[j];
          } else {
#pragma unroll
            for (int r = 0; r < 4; ++r) sv[j][b % NB][r] = cb == b / NB ? acc[j][r] : sv[j][b % NB][r];
          }
        }
      }
      const int tg = 16 * NB * cb + 4 * g;  // the lane's first token of the tile
#pragma unroll
      for (int k = 0; k < NB; ++k) {
        const ba_v4f nk4 = *reinterpret_cast<const ba_v4f*>(snorm + tg + 16 * k);
#pragma unroll
        for (int j = 0; j < NGR; ++j)
#pragma unroll
          for (int r = 0; r < 4; ++r) sv[j][k][r] *= nk4[r];
      }
      if (mods) {  // to the log2 domain, capped and biased
#pragma unroll
        for (int j = 0; j < NGR; ++j) {
          const float d0 = (float)(p0 + tg - qpos[j]);
#pragma unroll
          for (int k = 0; k < NB; ++k)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
              float y = sv[j][k][r] * kinv[j];
              if (a.cap2 != 0.f) y = ba_softcap<PREC>(y, a.cap2, a.cap2_inv);
              sv[j][k][r] = fmaf(slope[j], d0 + (float)(16 * k + r), y);
            }
        }
      }
      if (mask) {
#pragma unroll
        for (int j = 0; j < NGR; ++j) {
          const int rlo = lo[j] - p0 - tg, rhi = hi[j] - p0 - tg;
#pragma unroll
          for (int k = 0; k < NB; ++k)
#pragma unroll
            for (int r = 0; r < 4; ++r)
              sv[j][k][r] = 16 * k + r >= rlo && 16 * k + r < rhi ? sv[j][k][r] : -INFINITY;
        }
      }

      // ---- online softmax (log2 domain); weights times value norms as fp16
      ba_v4f nv4[NB];
#pragma unroll
      for (int k = 0; k < NB; ++k) nv4[k] = *reinterpret_cast<const ba_v4f*>(snorm + 64 + tg + 16 * k);
      ba_v8h bh[NGR][2], bl[PREC ? NGR : 1][2];
#pragma unroll
      for (int j = 0; j < NGR; ++j) {
        float mx = -INFINITY;
#pragma unroll
        for (int k = 0; k < NB; ++k)
#pragma unroll
          for (int r = 0; r < 4; ++r) mx = fmaxf(mx, sv[j][k][r]);
        mx = ba_max4(mx);
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
        typedef _Float16 v4h __attribute__((ext_vector_type(4)));
        v4h ph[NB], pl[NB];
#pragma unroll
        for (int k = 0; k < NB; ++k)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            // results below 2^-126 flush to 0: nothing beside the running maximum's 1
            const float p = __builtin_amdgcn_exp2f(fmaf(sv[j][k][r], kin, -ms));
            l[j] += p;
            float v = p * nv4[k][r];
            if (mask) v = p == 0.f ? 0.f : v;  // another row's inf or NaN norm
            if constexpr (PREC) {
              _Float16 hv, lv;
              split_f16(v, hv, lv);
              ph[k][r] = hv;
              pl[k][r] = lv;
            } else {
              ph[k][r] = (_Float16)v;
            }
          }
        // the second products' operand: 16-token group b in half b % 2 of part b / 2
        const v4h zero = {(_Float16)0.f, (_Float16)0.f, (_Float16)0.f, (_Float16)0.f};
#pragma unroll
        for (int b = 0; b < 4; ++b) {
          const bool mine = RW == 16 || cb == b / NB;
          const v4h x = mine ? ph[b % NB] : zero;
#pragma unroll
          for (int r = 0; r < 4; ++r) bh[j][b >> 1][4 * (b & 1) + r] = x[r];
          if constexpr (PREC) {
            const v4h y = mine ? pl[b % NB] : zero;
#pragma unroll
            for (int r = 0; r < 4; ++r) bl[j][b >> 1][4 * (b & 1) + r] = y[r];
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
            const uint8_t* q0 = vt + vaddr(t.vw[2 * s], nb);
            const uint8_t* q1 = vt + vaddr(t.vw[2 * s + 1], nb);
            const ba_u32x2 e0 = *reinterpret_cast<const ba_u32x2*>(q0), e1 = *reinterpret_cast<const ba_u32x2*>(q1);
            ah = ba_h8(e0.x, e0.y, e1.x, e1.y);
            if constexpr (PREC) {
              const ba_u32x2 f0 = *reinterpret_cast<const ba_u32x2*>(q0 + 128), f1 = *reinterpret_cast<const ba_u32x2*>(q1 + 128);
              al = ba_h8(f0.x, f0.y, f1.x, f1.y);
            }
          } else {
            const uint32_t vw = vword(s, nb);
            const uint8_t* q0 = vt + vaddr(vw, 0);
            const uint8_t* q1 = vt + vaddr(vw, 1);
            const uint8_t* q2 = vt + vaddr(vw, 2);
            const uint8_t* q3 = vt + vaddr(vw, 3);
            ah = ba_h8(*reinterpret_cast<const uint32_t*>(q0), *reinterpret_cast<const uint32_t*>(q1),
                       *reinterpret_cast<const uint32_t*>(q2), *reinterpret_cast<const uint32_t*>(q3));
            if constexpr (PREC)
              al = ba_h8(*reinterpret_cast<const uint32_t*>(q0 + 128), *reinterpret_cast<const uint32_t*>(q1 + 128),
                         *reinterpret_cast<const uint32_t*>(q2 + 128), *reinterpret_cast<const uint32_t*>(q3 + 128));
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

    if constexpr (NGR == 1) {  // three buffers, two tiles ahead; whole groups of three, then the rest
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
    } else if (nw > 0) {  // two buffers: the third would spill, and a tile takes longer here
      Tile r0, r1;
      load(0, r0);
      int i = 0;
      for (; i + 1 < nw; i += 2) {
        load(i + 1, r1);
        compute(i, r0);
        load(i + 2, r0);
        compute(i + 1, r1);
      }
      if (i < nw) compute(i, r0);
    }

    // ---- the piece's sums: over the row's lanes and, for few rows, its copies
    const float vinv = vs.inv() / vsc;  // powers of two
#pragma unroll
    for (int j = 0; j < NGR; ++j) {
      l[j] += __shfl_xor(l[j], 16, 64);
      l[j] += __shfl_xor(l[j], 32, 64);
      float f = vinv;
      if constexpr (RW < 16) {
        float M = m[j];
#pragma unroll
        for (int x = RW; x < 16; x <<= 1) M = fmaxf(M, __shfl_xor(M, x, 64));
        const float e = __builtin_amdgcn_exp2f(m[j] - (M == -INFINITY ? 0.f : M));
        m[j] = M;
        l[j] *= e;
        f *= e;
#pragma unroll
        for (int x = RW; x < 16; x <<= 1) l[j] += __shfl_xor(l[j], x, 64);
      }
#pragma unroll
      for (int nb = 0; nb < 4; ++nb) {
        o[j][nb] *= f;
        if constexpr (RW < 16) {
#pragma unroll
          for (int x = RW; x < 16; x <<= 1)
#pragma unroll
            for (int r = 0; r < 4; ++r) o[j][nb][r] += __shfl_xor(o[j][nb][r], x, 64);
        }
      }
      if (cb == 0 && row0 + 16 * j + cr <= lastrow) {
        const int64_t rowid = (int64_t)tok[j] * a.hq + qh[j];
        float* slot = ln.slots + ((int64_t)w * 2 + (ta == 0)) * ba_slot_floats(R);
        float* sums = whole ? ln.row_sums + rowid * 64 : slot + (16 * j + cr) * 64;
        float* st = whole ? ln.row_stats + rowid * 2 : slot + R * 64 + (16 * j + cr) * 2;
#pragma unroll
        for (int nb = 0; nb < 4; ++nb) *reinterpret_cast<ba_v4f*>(sums + 16 * nb + 4 * g) = o[j][nb];
        if (g == 0) {
          st[0] = m[j];
          st[1] = l[j];
        }
      }
    }
  }
}

template <int VB, bool SUB, bool PREC>
void ba_launch_kind(const BaArgs& a, int l, int rw, int groups, unsigned grid, hipStream_t st) {
  constexpr int N = ba_groups(PREC);
  const dim3 gr(grid), bl(kBaThreads);
  const BaLine& ln = a.line[l];
  if (groups > 1) hipLaunchKernelGGL((batch_attn_kernel<VB, SUB, PREC, 16, N>), gr, bl, 0, st, a, ln);
  else if (rw == 16) hipLaunchKernelGGL((batch_attn_kernel<VB, SUB, PREC, 16, 1>), gr, bl, 0, st, a, ln);
  else if (rw == 8) hipLaunchKernelGGL((batch_attn_kernel<VB, SUB, PREC, 8, 1>), gr, bl, 0, st, a, ln);
  else hipLaunchKernelGGL((batch_attn_kernel<VB, SUB, PREC, 4, 1>), gr, bl, 0, st, a, ln);
}

}  // namespace

template <int VB>
void ba_launch(const BaArgs& a, int l, bool sub, bool prec, int rw, int groups, unsigned grid, hipStream_t st) {
  if (sub && prec) ba_launch_kind<VB, true, true>(a, l, rw, groups, grid, st);
  else if (sub) ba_launch_kind<VB, true, false>(a, l, rw, groups, grid, st);
  else if (prec) ba_launch_kind<VB, false, true>(a, l, rw, groups, grid, st);
  else ba_launch_kind<VB, false, false>(a, l, rw, groups, grid, st);
}

}  // namespace tq
