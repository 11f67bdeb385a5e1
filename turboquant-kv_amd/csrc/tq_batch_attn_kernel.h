// tq_batch_attn_kernel.h -- the main kernel described in tq_batch_attn.h, and ba_launch<VB>.
#pragma once

#include "tq_batch_attn.h"

namespace tq {
namespace {

// LDS: key table, value table, each wave's norms of a tile.  An entry has 256 bytes of copies, or
// (PREC) 128 of its hi part, and its lo part's kBaLo bytes from them: in the second half of the
// eighth entry on (the last keys' in the first value entries').  Nearer, the compiler would read
// both parts with one instruction, side by side, and move them to the operands they belong to:
// 96 moves a tile.
constexpr int kBaVTab = 65536;
constexpr int kBaLo = 2048 + 128;
constexpr int kBaNorms = 131072 + 2048;  // [waves][2][64] floats

// Weights reach 2^kBaSlack before their reference moves; norms are scaled down by as much less one.
constexpr float kBaSlack = 4.f, kBaNormDown = 0.125f;

__device__ __forceinline__ ba_v8h ba_h8(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  ba_u32x4 t = {a, b, c, d};
  return __builtin_bit_cast(ba_v8h, t);
}

// cap2 tanh(z) of x = 2 z log2(e), in two forms.  Small: z times a polynomial in z^2 -- the odd
// series up to z^11 (the next term is 6e-10 relative at |z| = 0.3), or, for bf16 queries, up to
// z^5 with the z^7 term economized over |z| <= 0.3 (3e-6 relative): four instructions.  Any:
// tanh z = 1 - 2 / (1 + e^(2 z)), exact at both ends (the exponential overflows to inf or
// vanishes), whose absolute error of about 2^-23 is cap2 2^-23 in the score.
constexpr float kBaSmallCap = 0.3f * 2.885390081777927f;
template <bool PREC>
__device__ __forceinline__ float ba_softcap_small(float x, float cap2) {
  constexpr float h = 0.34657359027997264f;  // z / x
  const float w = x * x;
  if constexpr (PREC) {
    constexpr float h2 = h * h, h4 = h2 * h2;
    float p = fmaf(w, -0.00886323552990f * h4 * h4 * h2, 0.0218694885361f * h4 * h4);
    p = fmaf(w, p, -0.0539682539683f * h4 * h2);
    p = fmaf(w, p, 0.133333333333f * h4);
    p = fmaf(w, p, -0.333333333333f * h2);
    const float y = x * (h * cap2);
    return fmaf(y * w, p, y);
  } else {
    const float k = h * cap2;
    const float p = fmaf(w, k * (0.126048f * h * h * h * h), k * (-0.333087f * h * h));
    return x * fmaf(w, p, k * 0.9999988f);
  }
}
template <bool PREC>
__device__ __forceinline__ float ba_softcap_any(float x, float cap2) {
  const float big = fmaf(-2.f * cap2, __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(x)), cap2);
  return PREC && fabsf(x) < kBaSmallCap ? ba_softcap_small<true>(x, cap2) : big;
}

// The least (greatest) of v over RW neighbouring lanes, the rows of a group of columns; uniform.
template <int RW>
__device__ __forceinline__ int ba_rows_min(int v) {
#pragma unroll
  for (int o = RW / 2; o >= 1; o >>= 1) v = min(v, __shfl_xor(v, o, 64));
  return __builtin_amdgcn_readfirstlane(v);
}
template <int RW>
__device__ __forceinline__ int ba_rows_max(int v) {
#pragma unroll
  for (int o = RW / 2; o >= 1; o >>= 1) v = max(v, __shfl_xor(v, o, 64));
  return __builtin_amdgcn_readfirstlane(v);
}

// Loads through a raw buffer resource: a lane's 32-bit offset plus a scalar one, no vector
// address arithmetic.
template <typename T>
__device__ __forceinline__ T ba_load(__amdgpu_buffer_rsrc_t rs, uint32_t lane_off, uint32_t off) {
  if constexpr (sizeof(T) == 4) return __builtin_bit_cast(T, __builtin_amdgcn_raw_buffer_load_b32(rs, lane_off, off, 0));
  else if constexpr (sizeof(T) == 8) return __builtin_bit_cast(T, __builtin_amdgcn_raw_buffer_load_b64(rs, lane_off, off, 0));
  else return __builtin_bit_cast(T, __builtin_amdgcn_raw_buffer_load_b128(rs, lane_off, off, 0));
}

// fp16 hi and lo parts of a (low half) and b.  (Each is pinned as one fp32 value first: a product
// folded into both conversions would be rounded apart.)
__device__ __forceinline__ void ba_split(float a, float b, uint32_t& hi, uint32_t& lo) {
  typedef float v2f __attribute__((ext_vector_type(2)));
  typedef _Float16 v2h __attribute__((ext_vector_type(2)));
  asm("" : "+v"(a), "+v"(b));
  const v2h h = __builtin_convertvector((v2f){a, b}, v2h);
  hi = __builtin_bit_cast(uint32_t, h);
  lo = __builtin_bit_cast(uint32_t, __builtin_convertvector((v2f){a - (float)h[0], b - (float)h[1]}, v2h));
}

// The larger of two numbers in one instruction (fmaxf first quiets operands it cannot see
// through); NaN yields the other one.
__device__ __forceinline__ float ba_max(float a, float b) {
  float r;
  asm("v_max_f32 %0, %1, %2" : "=v"(r) : "v"(a), "v"(b));
  return r;
}

// The larger of x over the lanes c, c + 16, c + 32, c + 48.
__device__ __forceinline__ float ba_max4(float x) {
  const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  x = ba_max(__uint_as_float(a[0]), __uint_as_float(a[1]));
  const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return ba_max(__uint_as_float(b[0]), __uint_as_float(b[1]));
}

// Builds the tables in LDS from the entries that the preparing kernel made; every wave calls it
// once, after asking for its first item's data.
template <int VB, bool PREC>
__device__ __forceinline__ void ba_build_tables(const BaArgs& a, uint8_t* smem) {
  const int tid = threadIdx.x;
  const int e = tid & 255;  // threads t, t + 256, .. write entry t's copies in turn, 16 bytes each
  const BaEntry x = a.entries[e];
#pragma unroll
  for (int k = tid >> 8; k < 16; k += kBaWaves / 4) {
    // rotated by the entry so that a wave's stores spread over the banks
    const int q = (k + e) & 15;
    const bool second = PREC && q >= 8;
    const uint32_t kx = second ? x.klo : x.khi;
    const uint32_t v0 = second ? x.vlo[0] : x.vhi[0], v1 = VB == 2 ? (second ? x.vlo[1] : x.vhi[1]) : v0;
    const int at = e * 256 + 16 * q + (second ? kBaLo - 128 : 0);
    *reinterpret_cast<ba_u32x4*>(smem + at) = (ba_u32x4){kx, kx, kx, kx};
    *reinterpret_cast<ba_u32x4*>(smem + kBaVTab + at) = (ba_u32x4){v0, v1, v0, v1};
  }
  __syncthreads();
}

// A wave's piece of line `ln`.  RW rows of 16 columns (16 / RW copies share a tile's tokens), NGR
// groups of columns; WIDE: pools of 4 GB and more, whose rows need 64-bit addresses; MODS: scores
// may be capped or biased.
template <int VB, bool SUB, bool PREC, int RW, int NGR, bool WIDE, bool MODS>
__device__ __forceinline__ void ba_piece(const BaArgs& a, const BaLine& ln, uint8_t* smem, int w, bool& built) {
#pragma clang fp contract(off)
  static_assert(NGR == 1 || RW == 16, "groups of columns hold 16 rows each");
  constexpr int NB = RW / 4;       // 16-token groups whose scores a lane keeps
  constexpr int R = RW * NGR;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int c = lane & 15, g = lane >> 4;
  const int cb = c / RW, cr = c % RW;  // the column's copy and row
  const int hkv = a.hkv, G = a.G;
  int item = __builtin_amdgcn_readfirstlane(ln.work[w]);
  if (item < 0) return;
  auto uniform64 = [](int64_t x) {
    return (int64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)x) |
           (int64_t)__builtin_amdgcn_readfirstlane((int)(x >> 32)) << 32;
  };
  BaItem it = ln.items[item];
  const int64_t chunk = uniform64(ln.head->chunk), total = uniform64(ln.head->total);
  const float vsc_inv = a.entries[0].vsc_inv;  // a power of two
  // this lane's copy of an entry's hi part
  const uint32_t koff = PREC ? 4u * (lane & 31) : 4u * lane;
  // (byte 1: the value table's 64 KB, byte 2 of its addresses)
  const uint32_t voff = (VB == 2 ? (PREC ? 8u * (lane & 15) : 8u * (lane & 31)) : koff) | 0x100u;
  static_assert(kBaVTab == 0x10000, "value table");
  // address of byte i of w: entry i * 256 + copy
  auto kaddr = [&](uint32_t w, int i) -> uint32_t {
    return __builtin_amdgcn_perm(koff, w, 0x0c0c0004u | ((uint32_t)i << 8));
  };
  const uint32_t vsel = lane & 1 ? 0x07060302u : 0x05040100u;  // a lane's half of shared words
  auto vaddr = [&](uint32_t w, int i) -> uint32_t {
    return __builtin_amdgcn_perm(voff, w, 0x0c050004u | ((uint32_t)i << 8));
  };


  const int bsl = a.bs_log2;
  float* const snorm = reinterpret_cast<float*>(smem + kBaNorms) + wave * 128;
  const __amdgpu_buffer_rsrc_t krs = buf_rsrc(a.kpairs, 0xFFFFFFFFu), vrs = buf_rsrc(a.vtiles, 0xFFFFFFFFu);
  const __amdgpu_buffer_rsrc_t knrs = buf_rsrc(a.knorms, 0xFFFFFFFFu), vnrs = buf_rsrc(a.vnorms, 0xFFFFFFFFu);
  int64_t pos = (int64_t)w * chunk;
  const int64_t end = min(pos + chunk, total);

  while (pos < end) {  // (item, head)s of the piece
    const int t0 = __builtin_amdgcn_readfirstlane(it.t0), nt = __builtin_amdgcn_readfirstlane(it.nt);
    const int tok0 = __builtin_amdgcn_readfirstlane(it.tok0), row0 = __builtin_amdgcn_readfirstlane(it.row0);
    const int lastrow = __builtin_amdgcn_readfirstlane(it.nrows) - 1;
    const int table = __builtin_amdgcn_readfirstlane(it.table);
    const int cost = nt + kBaOver;
    const int64_t start = uniform64(it.start);
    const int h = (int)ba_div(pos - start, cost);
    const int off = (int)(pos - start - (int64_t)h * cost);
    const int n = (int)min<int64_t>(cost - off, end - pos);
    const int ta = (int)ba_tiles(off), tb = (int)ba_tiles(off + n);
    const bool whole = tb - ta == nt && (nt > 0 || off == 0);
    pos += n;
    const int it_lo = __builtin_amdgcn_readfirstlane(it.lo), it_hi = __builtin_amdgcn_readfirstlane(it.hi);
    const bool next = off + n == cost && h == hkv - 1 && pos < end;
    if (!whole && ta == tb) {
      if (next) it = ln.items[++item];
      continue;
    }

    const int k0 = t0 + ta, nw = tb - ta;  // tiles of the piece
    // Pool rows of 16 tiles' 16-token groups at a time (lane 4 i + b: tile i's group b), the next
    // 16 tiles' block ids requested while these are used.
    const int32_t* btab = a.block_tables + (int64_t)table * a.table_stride;
    auto load_ids = [&](int chunk16) -> uint32_t {
      const int i = min(chunk16 * 16 + (lane >> 2), nw - 1);
      const int64_t tb = ((int64_t)(k0 + i) << 6) + 16 * (lane & 3);
      const int bi = (int)min<int64_t>(tb >> bsl, (int64_t)a.max_blocks - 1);
      return (uint32_t)btab[bi];
    };
    using row_t = std::conditional_t<WIDE, uint64_t, uint32_t>;
    auto pool_row = [&](uint32_t id, int chunk16) -> row_t {
      const uint32_t tb = ((uint32_t)(k0 + chunk16 * 16 + (lane >> 2)) << 6) + 16u * (lane & 3);
      return (((row_t)min(id, a.num_blocks - 1u) * (uint32_t)hkv + (uint32_t)h) << bsl) + (tb & ((1u << bsl) - 1u));
    };
    uint32_t ids_next = 0;
    if (nw > 0) ids_next = load_ids(0);

    auto place_of = [&](int j, int& tok, int& qh) {
      const int row = min(row0 + 16 * j + cr, lastrow), ti = row / G;
      tok = tok0 + ti;
      qh = h * G + (row - ti * G);
    };
    // ---- rows: group j's column c holds row row0 + 16 j + cr (past the end: the last)
    int lo[NGR], hi[NGR], qpos[NGR];
    float slope[NGR];
    int qe[NGR], qtop = INT_MIN;
    ba_v8h qhi[NGR][2], qlo[PREC ? NGR : 1][2];
#pragma unroll
    for (int j = 0; j < NGR; ++j) {
      int tok, qh;
      place_of(j, tok, qh);
      const BaToken t = a.tokens[tok];
      lo[j] = max(t.lo, it_lo);
      hi[j] = min(t.hi, it_hi);
      qpos[j] = t.pos;
      const int64_t rowid = (int64_t)tok * a.hq + qh;
      qe[j] = a.qexp[rowid];
      qtop = max(qtop, qe[j]);
      slope[j] = MODS && a.slopes ? a.slopes[qh] * 1.4426950408889634f : 0.f;
#pragma unroll
      for (int s = 0; s < 2; ++s) {  // dims 16 g + 8 s ..
        qhi[j][s] = *reinterpret_cast<const ba_v8h*>(a.qhi + rowid * 64 + 16 * g + 8 * s);
        if constexpr (PREC) qlo[j][s] = *reinterpret_cast<const ba_v8h*>(a.qlo + rowid * 64 + 16 * g + 8 * s);
      }
    }
    // One power of two for all the wave's rows, so that it goes with the key norms: shorter queries
    // are scaled down to the longest's.  Errors stay under 2^-22 (bf16 queries: 2^-11) of a row's
    // own length down to lengths 2^-17 (2^-28) of the longest row's.
    qtop = ba_rows_max<RW>(qtop);
#pragma unroll
    for (int j = 0; j < NGR; ++j)
      if (__any(qe[j] != qtop)) {
        const float f = __builtin_amdgcn_ldexpf(1.f, max(qe[j] - qtop, -100));
#pragma unroll
        for (int s = 0; s < 2; ++s)
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            qhi[j][s][i] = (_Float16)((float)qhi[j][s][i] * f);
            if constexpr (PREC) qlo[j][s][i] = (_Float16)((float)qlo[j][s][i] * f);
          }
      }
    // the key norms' factor: scores in the log2 domain, or what ba_softcap takes
    const float kscale = __builtin_amdgcn_ldexpf(MODS && a.cap2 != 0.f ? 2.885390081777927f * a.cap2_inv : 1.f, qtop);
    int lo_min = INT_MAX, lo_max = 0, hi_min = INT_MAX, hi_max = 0;
#pragma unroll
    for (int j = 0; j < NGR; ++j) {
      lo_min = min(lo_min, lo[j]);
      lo_max = max(lo_max, lo[j]);
      hi_min = min(hi_min, hi[j]);
      hi_max = max(hi_max, hi[j]);
    }
    lo_min = ba_rows_min<RW>(lo_min);
    lo_max = ba_rows_max<RW>(lo_max);
    hi_min = ba_rows_min<RW>(hi_min);
    hi_max = ba_rows_max<RW>(hi_max);

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

    constexpr int NV = VB == 2 ? 4 : (SUB ? 8 : 2 * VB);
    struct Tile {
      ba_u32x2 kw[4];
      float nk, nv;
      uint32_t vw[NV];
    };
    row_t rows16 = 0;
    // i: the wave's i-th tile, asked for in order (a repeated last one excepted)
    auto load = [&](int i, Tile& t) {
      if ((i & 15) == 0 && i < nw) {
        rows16 = pool_row(ids_next, i >> 4);
        ids_next = load_ids((i >> 4) + 1);
      }
      const int from = 4 * (min(i, nw - 1) & 15);
      auto row_of = [&](int b) -> row_t {  // of 16-token group b
        row_t r = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)rows16, from + b);
        if constexpr (WIDE) r |= (row_t)(uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(rows16 >> 32), from + b) << 32;
        return r;
      };
      // T at `extra` bytes plus a lane's offset into the bytes of row `r` of a pool
      auto at = [&](auto tag, const void* pool, __amdgpu_buffer_rsrc_t rs, uint32_t lane_off, row_t r, int bytes, int extra = 0) {
        using T = decltype(tag);
        if constexpr (WIDE)
          return ba_load<T>(buf_rsrc(static_cast<const uint8_t*>(pool) + r * bytes + extra, 0xFFFFFFFFu), lane_off, 0);
        else
          return ba_load<T>(rs, lane_off + extra, (uint32_t)r * bytes);
      };
      row_t row[4];
#pragma unroll
      for (int b = 0; b < 4; ++b) row[b] = SUB || b == 0 ? row_of(b) : row[0] + 16 * b;
      if constexpr (SUB) {  // a lane's token: number c of group g
        const int src = 4 * (from + g);
        uint32_t lo32 = (uint32_t)__builtin_amdgcn_ds_bpermute(src, (int)(uint32_t)rows16);
        if constexpr (WIDE) {
          const row_t r = lo32 | (row_t)(uint32_t)__builtin_amdgcn_ds_bpermute(src, (int)(uint32_t)(rows16 >> 32)) << 32;
          t.nk = a.knorms[r + (uint32_t)c];
          t.nv = a.vnorms[r + (uint32_t)c];
        } else {
          t.nk = ba_load<float>(knrs, 4u * (lo32 + (uint32_t)c), 0);
          t.nv = ba_load<float>(vnrs, 4u * (lo32 + (uint32_t)c), 0);
        }
      } else {
        t.nk = at(float{}, a.knorms, knrs, 4u * lane, row[0], 4);
        t.nv = at(float{}, a.vnorms, vnrs, 4u * lane, row[0], 4);
      }
#pragma unroll
      for (int b = 0; b < 4; ++b) t.kw[b] = at(ba_u32x2{}, a.kpairs, krs, 32u * c + 8u * g, row[b], 32);
      if constexpr (SUB) {
#pragma unroll
        for (int b = 0; b < 4; ++b) {
          if constexpr (VB == 2) {
            t.vw[b] = at(uint32_t{}, a.vtiles, vrs, 4u * lane, row[b], 8 * VB);
          } else if constexpr (VB == 4) {
            const ba_u32x2 x = at(ba_u32x2{}, a.vtiles, vrs, 8u * lane, row[b], 8 * VB);
            t.vw[2 * b] = x.x;
            t.vw[2 * b + 1] = x.y;
          } else {  // the 16-bit share comes with its neighbour's: vsel picks it
            t.vw[b] = at(uint32_t{}, a.vtiles, vrs, 4u * lane, row[b], 8 * VB);
            t.vw[4 + b] = at(uint32_t{}, a.vtiles, vrs, 4u * (lane >> 1), row[b], 8 * VB, 256);
          }
        }
      } else {
        const ba_u32x4 v = at(ba_u32x4{}, a.vtiles, vrs, 16u * lane, row[0], 8 * VB);
        t.vw[0] = v.x; t.vw[1] = v.y; t.vw[2] = v.z; t.vw[3] = v.w;
        if constexpr (VB == 3) {
          const ba_u32x2 v1 = at(ba_u32x2{}, a.vtiles, vrs, 8u * lane, row[0], 8 * VB, 1024);
          t.vw[4] = v1.x; t.vw[5] = v1.y;
        } else if constexpr (VB == 4) {
          const ba_u32x4 v1 = at(ba_u32x4{}, a.vtiles, vrs, 16u * lane, row[0], 8 * VB, 1024);
          t.vw[4] = v1.x; t.vw[5] = v1.y; t.vw[6] = v1.z; t.vw[7] = v1.w;
        }
      }
    };

    auto compute = [&](int i, const Tile& t) {
      const int p0 = (k0 + i) << 6;  // position of the tile's first token
      const bool mask = p0 < lo_max || p0 + 64 > hi_min;
      float nvl = t.nv;
      bool odd = false;  // a token that not all rows see has an inf or NaN norm
      if (__builtin_expect(mask, 0)) {
        // norms of tokens no row sees may be stale, even NaN
        nvl = p0 + lane >= lo_min && p0 + lane < hi_max ? t.nv : 0.f;
        odd = __any(!(fabsf(nvl) < INFINITY));
      }
      if (vs.over(fabsf(nvl) * vs.s)) {
        const float f = vs.rescale(fabsf(nvl));
#pragma unroll
        for (int j = 0; j < NGR; ++j)
#pragma unroll
          for (int nb = 0; nb < 4; ++nb) o[j][nb] *= f;
      }
      snorm[lane] = t.nk * kscale;
      // (weights are at most 2^kBaSlack: their products with norms stay below 2^15)
      if constexpr (PREC) snorm[64 + lane] = nvl * (vs.s * kBaNormDown);
      else reinterpret_cast<_Float16*>(snorm + 64)[lane] = (_Float16)(nvl * (vs.s * kBaNormDown));
      __builtin_amdgcn_wave_barrier();

      // value word helpers: VB 3 / 4, tile word i of half s, and the word whose bytes index
      // the pair entries of dim group nb
      auto tword = [&](int s, int i2) -> uint32_t {
        if constexpr (!SUB) {
          return t.vw[(VB == 4 ? 4 : 3) * s + i2];
        } else if constexpr (VB == 4) {
          return __builtin_amdgcn_perm(t.vw[2 * (2 * s + 1) + (i2 >> 1)], t.vw[2 * (2 * s) + (i2 >> 1)],
                                       (i2 & 1) ? 0x07060302u : 0x05040100u);
        } else {
          return i2 == 2 ? __builtin_amdgcn_perm(t.vw[4 + 2 * s + 1], t.vw[4 + 2 * s], vsel)
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


      // ---- scores: entry k of a lane is its copy's 16-token group NB cb + k
      ba_v4f sv[NGR][NB], all[NGR][4];
#pragma unroll
      for (int j = 0; j < NGR; ++j)
#pragma unroll
        for (int b = 0; b < 4; ++b) all[j][b] = (ba_v4f){0.f, 0.f, 0.f, 0.f};
      // (KB 16-token groups at a time, so that products of one sum do not follow each other)
      constexpr int KB = NGR == 1 ? 4 : 1;
#pragma unroll
      for (int b0 = 0; b0 < 4; b0 += KB) {
#pragma unroll
        for (int s = 0; s < 2; ++s) {
          ba_v8h ah[KB], al[PREC ? KB : 1];
#pragma unroll
          for (int b = 0; b < KB; ++b) {
            const uint32_t kw = t.kw[b0 + b][s];
            const uint8_t* p0a = smem + kaddr(kw, 0);
            const uint8_t* p1a = smem + kaddr(kw, 1);
            const uint8_t* p2a = smem + kaddr(kw, 2);
            const uint8_t* p3a = smem + kaddr(kw, 3);
            ah[b] = ba_h8(*reinterpret_cast<const uint32_t*>(p0a), *reinterpret_cast<const uint32_t*>(p1a),
                          *reinterpret_cast<const uint32_t*>(p2a), *reinterpret_cast<const uint32_t*>(p3a));
            if constexpr (PREC)
              al[b] = ba_h8(*reinterpret_cast<const uint32_t*>(p0a + kBaLo), *reinterpret_cast<const uint32_t*>(p1a + kBaLo),
                            *reinterpret_cast<const uint32_t*>(p2a + kBaLo), *reinterpret_cast<const uint32_t*>(p3a + kBaLo));
          }
#pragma unroll
          for (int p = 0; p < (PREC ? 3 : 1); ++p)
#pragma unroll
            for (int b = 0; b < KB; ++b)
#pragma unroll
              for (int j = 0; j < NGR; ++j)
                all[j][b0 + b] = __builtin_amdgcn_mfma_f32_16x16x32_f16(p == 2 ? al[PREC ? b : 0] : ah[b],
                                                                        p == 1 ? qlo[PREC ? j : 0][s] : qhi[j][s],
                                                                        all[j][b0 + b], 0, 0, 0);
        }
      }
#pragma unroll
      for (int j = 0; j < NGR; ++j)
#pragma unroll
        for (int b = 0; b < 4; ++b) {
          if (b / NB == 0) {
            sv[j][b] = all[j][b];
          } else {
#pragma unroll
            for (int r = 0; r < 4; ++r) sv[j][b % NB][r] = cb == b / NB ? all[j][b][r] : sv[j][b % NB][r];
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
      if (MODS && a.cap2 != 0.f) {  // most tiles hold no score near the cap
#pragma unroll
        for (int j = 0; j < NGR; ++j) {
          float far = 0.f;
#pragma unroll
          for (int k = 0; k < NB; ++k)
#pragma unroll
            for (int r = 0; r < 4; ++r) far = fmaxf(far, fabsf(sv[j][k][r]));
          if (__any(far >= kBaSmallCap)) {
            asm volatile("");
#pragma unroll
            for (int k = 0; k < NB; ++k)
#pragma unroll
              for (int r = 0; r < 4; ++r) sv[j][k][r] = ba_softcap_any<PREC>(sv[j][k][r], a.cap2);
          } else {
            asm volatile("");
#pragma unroll
            for (int k = 0; k < NB; ++k)
#pragma unroll
              for (int r = 0; r < 4; ++r) sv[j][k][r] = ba_softcap_small<PREC>(sv[j][k][r], a.cap2);
          }
        }
      }
      if (MODS && a.slopes) {
#pragma unroll
        for (int j = 0; j < NGR; ++j) {
          const float d0 = (float)(p0 + tg - qpos[j]);
#pragma unroll
          for (int k = 0; k < NB; ++k)
#pragma unroll
            for (int r = 0; r < 4; ++r) sv[j][k][r] = fmaf(slope[j], d0 + (float)(16 * k + r), sv[j][k][r]);
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
      ba_v4f nv4[PREC ? NB : 1];
      ba_u32x2 nvh[PREC ? 1 : NB];  // two fp16 a word
#pragma unroll
      for (int k = 0; k < NB; ++k) {
        if constexpr (PREC) nv4[k] = *reinterpret_cast<const ba_v4f*>(snorm + 64 + tg + 16 * k);
        else nvh[k] = *reinterpret_cast<const ba_u32x2*>(reinterpret_cast<const _Float16*>(snorm + 64) + tg + 16 * k);
      }
      ba_v8h bh[NGR][2], bl[PREC ? NGR : 1][2];
#pragma unroll
      for (int j = 0; j < NGR; ++j) {
        float mx = -INFINITY;
#pragma unroll
        for (int k = 0; k < NB; ++k)
#pragma unroll
          for (int r = 0; r < 4; ++r) mx = fmaxf(mx, sv[j][k][r]);
        // The weights' reference m[j] follows the maximum only when a score passes it by kBaSlack:
        // most tiles neither exchange maxima between lanes nor rescale.
        if (__any(mx > m[j] + kBaSlack)) {
          const float mn = ba_max4(ba_max(mx, m[j]));
          const float alpha = __builtin_amdgcn_exp2f(m[j] - (mn == -INFINITY ? 0.f : mn));
          l[j] *= alpha;
#pragma unroll
          for (int nb = 0; nb < 4; ++nb) o[j][nb] *= alpha;
          m[j] = mn;
        }
        const float ms = m[j] == -INFINITY ? 0.f : m[j];
        // weights times value norms, two fp16 a word: word q of group k holds tokens 2 q, 2 q + 1
        uint32_t ph[NB][2], pl[PREC ? NB : 1][2];
#pragma unroll
        for (int k = 0; k < NB; ++k)
#pragma unroll
          for (int q = 0; q < 2; ++q) {
            // results below 2^-126 flush to 0: nothing beside the running maximum's 1
            const float pa = __builtin_amdgcn_exp2f(sv[j][k][2 * q] - ms);
            const float pb = __builtin_amdgcn_exp2f(sv[j][k][2 * q + 1] - ms);
            if constexpr (PREC) {
              l[j] += pa + pb;
              ba_split(pa * nv4[k][2 * q], pb * nv4[k][2 * q + 1], ph[k][q], pl[k][q]);
            } else {  // the sum of the weights as they are rounded
              typedef float v2f __attribute__((ext_vector_type(2)));
              typedef _Float16 v2h __attribute__((ext_vector_type(2)));
              const v2h p = __builtin_convertvector((v2f){pa, pb}, v2h);
              l[j] = __builtin_amdgcn_fdot2(p, (v2h){(_Float16)1.f, (_Float16)1.f}, l[j], false);
              const uint32_t nv2 = nvh[k][q];  // (a bit cast of the vector's element itself reads element 0)
              ph[k][q] = __builtin_bit_cast(uint32_t, p * __builtin_bit_cast(v2h, nv2));
            }
          }
        if (__builtin_expect(odd, 0)) {  // rows that do not see it must not take 0 * inf
          asm volatile("");
#pragma unroll
          for (int k = 0; k < NB; ++k)
#pragma unroll
            for (int q = 0; q < 2; ++q) {
              const uint32_t keep = (sv[j][k][2 * q] == -INFINITY ? 0u : 0xFFFFu) |
                                    (sv[j][k][2 * q + 1] == -INFINITY ? 0u : 0xFFFF0000u);
              ph[k][q] &= keep;
              if constexpr (PREC) pl[k][q] &= keep;
            }
        }
        // the second products' operand: 16-token group b in half b % 2 of part b / 2
#pragma unroll
        for (int s = 0; s < 2; ++s) {
          uint32_t x[4], y[4];
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const int b = 2 * s + (q >> 1);
            const bool mine = RW == 16 || cb == b / NB;
            x[q] = mine ? ph[b % NB][q & 1] : 0u;
            if constexpr (PREC) y[q] = mine ? pl[b % NB][q & 1] : 0u;
          }
          bh[j][s] = ba_h8(x[0], x[1], x[2], x[3]);
          if constexpr (PREC) bl[j][s] = ba_h8(y[0], y[1], y[2], y[3]);
        }
      }
      // wait states between the conversions and the products that read them
      if constexpr (NGR == 3) {
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

      // ---- values (VN groups of 16 dims at a time, as above)
      constexpr int VN = NGR == 1 ? 4 : 1;
#pragma unroll
      for (int s = 0; s < 2; ++s) {
#pragma unroll
        for (int n0 = 0; n0 < 4; n0 += VN) {
          ba_v8h ah[VN], al[PREC ? VN : 1];
#pragma unroll
          for (int n = 0; n < VN; ++n) {
            const int nb = n0 + n;
            if constexpr (VB == 2) {
              const uint8_t* q0 = smem + vaddr(t.vw[2 * s], nb);
              const uint8_t* q1 = smem + vaddr(t.vw[2 * s + 1], nb);
              const ba_u32x2 e0 = *reinterpret_cast<const ba_u32x2*>(q0), e1 = *reinterpret_cast<const ba_u32x2*>(q1);
              ah[n] = ba_h8(e0.x, e0.y, e1.x, e1.y);
              if constexpr (PREC) {
                const ba_u32x2 f0 = *reinterpret_cast<const ba_u32x2*>(q0 + kBaLo);
                const ba_u32x2 f1 = *reinterpret_cast<const ba_u32x2*>(q1 + kBaLo);
                al[n] = ba_h8(f0.x, f0.y, f1.x, f1.y);
              }
            } else {
              const uint32_t vw = vword(s, nb);
              const uint8_t* q0 = smem + vaddr(vw, 0);
              const uint8_t* q1 = smem + vaddr(vw, 1);
              const uint8_t* q2 = smem + vaddr(vw, 2);
              const uint8_t* q3 = smem + vaddr(vw, 3);
              ah[n] = ba_h8(*reinterpret_cast<const uint32_t*>(q0), *reinterpret_cast<const uint32_t*>(q1),
                            *reinterpret_cast<const uint32_t*>(q2), *reinterpret_cast<const uint32_t*>(q3));
              if constexpr (PREC)
                al[n] = ba_h8(*reinterpret_cast<const uint32_t*>(q0 + kBaLo), *reinterpret_cast<const uint32_t*>(q1 + kBaLo),
                              *reinterpret_cast<const uint32_t*>(q2 + kBaLo), *reinterpret_cast<const uint32_t*>(q3 + kBaLo));
            }
          }
#pragma unroll
          for (int p = 0; p < (PREC ? 3 : 1); ++p)
#pragma unroll
            for (int n = 0; n < VN; ++n)
#pragma unroll
              for (int j = 0; j < NGR; ++j)
                o[j][n0 + n] = __builtin_amdgcn_mfma_f32_16x16x32_f16(p == 2 ? al[PREC ? n : 0] : ah[n],
                                                                      p == 1 ? bl[PREC ? j : 0][s] : bh[j][s],
                                                                      o[j][n0 + n], 0, 0, 0);
        }
      }
    };

    // Two buffers, one tile ahead, the SIMD's other wave covering the rest; single tokens of fp32 /
    // fp16 queries, whose tiles take longer, gain by a third (91 -> 87 us; bf16: 67 -> 69 us).
    constexpr bool THREE = PREC && RW < 16;
    Tile r0, r1;
    if (nw > 0) load(0, r0);
    if constexpr (THREE) {
      if (nw > 0) load(1, r1);
    }
    if (!built) {  // while the first tile is on its way
      ba_build_tables<VB, PREC>(a, smem);
      built = true;
    }
    if (nw > 0) {
      int i = 0;
      if constexpr (THREE) {
        Tile r2;
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
      } else {
        for (; i + 1 < nw; i += 2) {
          load(i + 1, r1);
          compute(i, r0);
          load(i + 2, r0);
          compute(i + 1, r1);
        }
        if (i < nw) compute(i, r0);
      }
    }

    if (next) it = ln.items[++item];
    // ---- the piece's sums: over the row's lanes and, for few rows, its copies
    const float vinv = vs.inv() * vsc_inv * (1.f / kBaNormDown);
#pragma unroll
    for (int j = 0; j < NGR; ++j) {
      l[j] += __shfl_xor(l[j], 16, 64);
      l[j] += __shfl_xor(l[j], 32, 64);
      float f = vinv;
      const bool done = NGR > 1 && whole && a.direct;
      if constexpr (NGR > 1) {
        if (done) {  // (sums over the weights' total: at most 2^11 in the norms' scale)
          const float inv = l[j] == 0.f ? 0.f : 1.f / l[j];
          ba_v4f x[4], out[4];
#pragma unroll
          for (int nb = 0; nb < 4; ++nb) x[nb] = o[j][nb] * inv;
          ba_rotate_back<PREC>(a.vrot16, x, lane, out);
          if (row0 + 16 * j + cr <= lastrow) {
            int tok, qh;
            place_of(j, tok, qh);
#pragma unroll
            for (int ob = 0; ob < 4; ++ob) ba_store(a, tok, qh, 16 * ob + 4 * g, out[ob] * vinv);
            if (a.lse && g == 0) a.lse[(int64_t)tok * a.hq + qh] = ba_lse(m[j], l[j]);
          }
        }
      }
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
        if (!done) o[j][nb] *= f;
        if constexpr (RW < 16) {
#pragma unroll
          for (int x = RW; x < 16; x <<= 1)
#pragma unroll
            for (int r = 0; r < 4; ++r) o[j][nb][r] += __shfl_xor(o[j][nb][r], x, 64);
        }
      }
      if (!done && cb == 0 && row0 + 16 * j + cr <= lastrow) {
        int tok, qh;
        place_of(j, tok, qh);
        const int64_t rowid = (int64_t)tok * a.hq + qh;
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

// Line 0 alone (PAIR: line 1, whose items hold many rows, before it: a wave goes on with its
// piece of the sequences' line while others still read prefixes).
template <int VB, bool SUB, bool PREC, int RW, int NGR, bool WIDE, bool PAIR, bool MODS>
__global__ __launch_bounds__(64 * kBaWaves, kBaWaves / 4) void batch_attn_kernel(BaArgs a) {
  __shared__ __attribute__((aligned(16))) uint8_t smem[kBaNorms + kBaWaves * 512];
  // Neighbouring pieces on one XCD (workgroup w runs on XCD w % 8): rows of one prefix read the
  // same tiles there, and adjacent KV heads of a 16-token block share lines of norms.  Few
  // pieces spread over the workgroups.
  const unsigned grid = gridDim.x;
  const unsigned blk = grid % 8 == 0 ? (blockIdx.x % 8) * (grid / 8) + blockIdx.x / 8 : blockIdx.x;
  const int w = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6)) * (int)grid + (int)blk;
  bool built = false;
  if constexpr (PAIR) {
    // Where both lines' pieces are few, line 0's begin behind line 1's, so that no wave takes one
    // of each: 16 requests over 2048 shared tokens 14.6 -> 11.5 us.
    const int waves = a.line[0].waves;
    const int n1 = a.line[1].head->pieces, n0 = a.line[0].head->pieces;
    const int skip = n1 + n0 <= waves ? n1 : 0;
    bool busy = false;
#pragma unroll
    for (int k = 0; k < kBaWaves; ++k) {
      const int x = k * (int)grid + (int)blk;
      busy |= x < n1 || x - skip < n0;
    }
    if (!busy) return;
    ba_piece<VB, SUB, PREC, 16, ba_groups(PREC, true), WIDE, MODS>(a, a.line[1], smem, w, built);
    ba_piece<VB, SUB, PREC, RW, NGR, WIDE, MODS>(a, a.line[0], smem, w < skip ? w + waves - skip : w - skip, built);
  } else {
    // (a workgroup's first piece: where it lies behind the line's end, all do)
    if (a.line[0].work[blk] < 0) return;
    ba_piece<VB, SUB, PREC, RW, NGR, WIDE, MODS>(a, a.line[0], smem, w, built);
  }
  if (!built) ba_build_tables<VB, PREC>(a, smem);
}

template <int VB, bool SUB, bool PREC, bool WIDE, bool PAIR>
void ba_launch_kind(const BaArgs& a, int rw, int groups, unsigned grid, hipStream_t st) {
  const dim3 gr(grid), bl(64 * kBaWaves);
  // Kernels of many rows come without the code of caps and biases too, whose registers they miss:
  // causal prompts 412 -> 391 us.
  constexpr int N = ba_groups(PREC, PAIR);
  const bool mods = a.cap2 != 0.f || a.slopes;
  if (groups > 1 && mods) hipLaunchKernelGGL((batch_attn_kernel<VB, SUB, PREC, 16, N, WIDE, PAIR, true>), gr, bl, 0, st, a);
  else if (groups > 1) hipLaunchKernelGGL((batch_attn_kernel<VB, SUB, PREC, 16, N, WIDE, PAIR, false>), gr, bl, 0, st, a);
  else if (rw == 16) hipLaunchKernelGGL((batch_attn_kernel<VB, SUB, PREC, 16, 1, WIDE, PAIR, true>), gr, bl, 0, st, a);
  else if (rw == 8) hipLaunchKernelGGL((batch_attn_kernel<VB, SUB, PREC, 8, 1, WIDE, PAIR, true>), gr, bl, 0, st, a);
  else hipLaunchKernelGGL((batch_attn_kernel<VB, SUB, PREC, 4, 1, WIDE, PAIR, true>), gr, bl, 0, st, a);
}

template <int VB, bool SUB, bool PAIR>
void ba_launch_lines(const BaArgs& a, bool wide, bool prec, int rw, int groups, unsigned grid, hipStream_t st) {
  if (wide && prec) ba_launch_kind<VB, SUB, true, true, PAIR>(a, rw, groups, grid, st);
  else if (wide) ba_launch_kind<VB, SUB, false, true, PAIR>(a, rw, groups, grid, st);
  else if (prec) ba_launch_kind<VB, SUB, true, false, PAIR>(a, rw, groups, grid, st);
  else ba_launch_kind<VB, SUB, false, false, PAIR>(a, rw, groups, grid, st);
}

}  // namespace

template <int VB, bool SUB>
void ba_launch(const BaArgs& a, bool pair, bool wide, bool prec, int rw, int groups, unsigned grid, hipStream_t st) {
  if (pair) ba_launch_lines<VB, SUB, true>(a, wide, prec, rw, groups, grid, st);
  else ba_launch_lines<VB, SUB, false>(a, wide, prec, rw, groups, grid, st);
}

}  // namespace tq
