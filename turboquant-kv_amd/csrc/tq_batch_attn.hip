// tq_batch_attn.hip -- entry points of the ragged batch's attention (tq_batch_attn.h): the choice
// of kernels, the workspace, and the kernel that joins the partial results.

#include "tq_batch_attn.h"

#include <algorithm>

namespace tq {
namespace {

// Where a launch over the groups left its partial results.
struct BaPrefix {
  const float* slots;
  const BaHead* head;
  const BaItem* items;
  const int32_t* seg_item;
  const float* row_sums;
  const float* row_stats;
  int max_items;
  int rows;  // of an item
};

// Joins the partial results of 16 rows: those of an item cut between workgroups and, with
// groups, the item's own and its group's.  The four waves take the sources in turn, then a
// wave each rotates a quarter of the result's dims.  A row's sums of one source are 256
// consecutive bytes; latency bounds it (a few microseconds).
__global__ __launch_bounds__(256) void batch_combine_kernel(BaArgs a, BaPrefix p, int rows, int with_groups) {
#pragma clang fp contract(off)
  __shared__ __attribute__((aligned(16))) float sums_s[4][16][68];
  __shared__ float stat_s[4][16][2];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int c = lane & 15, g = lane >> 4;
  const int ngr = rows / 16;
  const int j = (int)(blockIdx.x % (unsigned)ngr);
  const int h = (int)(blockIdx.x / (unsigned)ngr % (unsigned)a.hkv);
  const int item = (int)(blockIdx.x / (unsigned)ngr / (unsigned)a.hkv);
  if (item >= a.head->n_items) return;
  const BaItem it = a.items[item];
  const int64_t chunk = a.head->chunk, start = it.start + (int64_t)h * it.cost;
  const int64_t w0 = start / chunk, w1 = (start + it.cost - 1) / chunk;
  const bool cut = w1 > w0;
  if (!with_groups && !cut) return;  // written by its workgroup
  const BaSeg sg = ba_segment(a, it.seg, rows);
  const int nrows = sg.ntok * a.G, irow = it.rt * rows + 16 * j;
  if (irow >= nrows) return;
  const int row = min(irow + c, nrows - 1);
  const int ti = row / a.G, tok = sg.tok0 + ti, qh = h * a.G + (row - ti * a.G);
  const int64_t rowid = (int64_t)tok * a.hq + qh;
  const int ns = cut ? (int)(w1 - w0) + 1 : 1;
  // the row's sources of its group's launch
  int np = 0, prow = 0;
  int64_t p0 = 0;
  bool pcut = false;
  if (with_groups && it.seg < a.B && a.n_groups > 0) {
    const int gi = ba_last(a.n_groups, it.seg, [&](int i) { return a.group_start[i]; });
    const int b0 = a.group_start[gi], b1 = min(a.group_start[gi + 1], a.B);
    if (b0 >= 0 && it.seg >= b0 && it.seg < b1 && a.shared[gi] > 0) {
      const int t0 = ba_qs(a, b0), t1 = ba_qs(a, b1);
      if (tok >= t0 && tok < t1) {
        const int64_t ro = (int64_t)(tok - t0) * a.G + (qh - h * a.G);
        const BaItem pi = p.items[min(p.seg_item[gi] + (int)(ro / p.rows), p.max_items - 1)];
        const int64_t pc = p.head->chunk, ps = pi.start + (int64_t)h * pi.cost;
        prow = (int)(ro % p.rows);
        p0 = ps / pc;
        const int64_t p1 = (ps + pi.cost - 1) / pc;
        pcut = p1 > p0;
        np = (int)(p1 - p0) + 1;
      }
    }
  }
  int most = ns + np;
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) most = max(most, __shfl_xor(most, o, 64));
  float m = -INFINITY, l = 0.f;
  ba_v4f o4[4];
#pragma unroll
  for (int nb = 0; nb < 4; ++nb) o4[nb] = (ba_v4f){0.f, 0.f, 0.f, 0.f};
  for (int i = wave; i < most; i += 4) {
    const float *sums, *st;
    if (i >= ns + np) continue;
    if (i < ns) {
      const float* s = a.slots + ((w0 + i) * 2 + (i == 0)) * ba_slot_floats(rows);
      sums = cut ? s + (16 * j + c) * 64 : a.row_sums + rowid * 64;
      st = cut ? s + rows * 64 + (16 * j + c) * 2 : a.row_stats + rowid * 2;
    } else {
      const int k = i - ns;
      const float* s = p.slots + ((p0 + k) * 2 + (k == 0)) * ba_slot_floats(p.rows);
      sums = pcut ? s + prow * 64 : p.row_sums + rowid * 64;
      st = pcut ? s + p.rows * 64 + prow * 2 : p.row_stats + rowid * 2;
    }
    const float mi = st[0], li = st[1];
    const float mn = fmaxf(m, mi), ms = mn == -INFINITY ? 0.f : mn;
    const float fa = __builtin_amdgcn_exp2f(m - ms), fb = __builtin_amdgcn_exp2f(mi - ms);
    m = mn;
    l = l * fa + li * fb;
#pragma unroll
    for (int nb = 0; nb < 4; ++nb)
      o4[nb] = o4[nb] * fa + *reinterpret_cast<const ba_v4f*>(sums + 16 * nb + 4 * g) * fb;
  }
  float rv[16];  // R_v's entries of this wave's 16 dims, requested before the barrier
#pragma unroll
  for (int nb = 0; nb < 4; ++nb)
#pragma unroll
    for (int r = 0; r < 4; ++r) rv[4 * nb + r] = a.vrot[(16 * nb + 4 * g + r) * 64 + 16 * wave + c];
#pragma unroll
  for (int nb = 0; nb < 4; ++nb) *reinterpret_cast<ba_v4f*>(&sums_s[wave][c][16 * nb + 4 * g]) = o4[nb];
  if (g == 0) {
    stat_s[wave][c][0] = m;
    stat_s[wave][c][1] = l;
  }
  __syncthreads();
  float M = -INFINITY, L = 0.f, f[4];
#pragma unroll
  for (int w = 0; w < 4; ++w) M = fmaxf(M, stat_s[w][c][0]);
  const float Ms = M == -INFINITY ? 0.f : M;
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    f[w] = __builtin_amdgcn_exp2f(stat_s[w][c][0] - Ms);
    L += stat_s[w][c][1] * f[w];
  }
  const float inv = L == 0.f ? 0.f : 1.f / L;
  ba_v4f acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int nb = 0; nb < 4; ++nb) {
    ba_v4f x = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < 4; ++w) x += *reinterpret_cast<const ba_v4f*>(&sums_s[w][c][16 * nb + 4 * g]) * f[w];
#pragma unroll
    for (int r = 0; r < 4; ++r) acc = __builtin_amdgcn_mfma_f32_16x16x4f32(rv[4 * nb + r], x[r] * inv, acc, 0, 0, 0);
  }
  if (irow + c >= nrows) return;
  if (it.seg < a.B || a.zero_tail) {
    const int64_t oa = (int64_t)tok * a.out_stride + qh * 64 + 16 * wave + 4 * g;
    if (a.q_dt == TQ_F32) {
      *reinterpret_cast<ba_v4f*>(static_cast<float*>(a.out) + oa) = acc;
    } else if (a.q_dt == TQ_BF16) {
      typedef __bf16 b4_t __attribute__((ext_vector_type(4)));
      *reinterpret_cast<b4_t*>(static_cast<uint16_t*>(a.out) + oa) = __builtin_convertvector(acc, b4_t);
    } else {
      typedef _Float16 h4_t __attribute__((ext_vector_type(4)));
      *reinterpret_cast<h4_t*>(static_cast<uint16_t*>(a.out) + oa) = __builtin_convertvector(acc, h4_t);
    }
  }
  if (a.lse && wave == 0 && g == 0)
    a.lse[rowid] = L == 0.f ? -INFINITY : (M + __builtin_amdgcn_logf(L)) * 0.6931471805599453f;
}

// Which kernels a call runs, and its workspace.
struct BaPlan {
  bool prec, rows;   // rows: the row kernel
  int groups, pgroups;  // row groups of a wave: sequences, prefix groups
  int64_t items, pitems;
  unsigned grid, pgrid;
  size_t slots, pslots, row_bytes, total;
};

constexpr size_t kBaHeadBytes = 256;

BaPlan ba_plan(tq_dtype q_dtype, int64_t n, int hq, int hkv, int64_t B, int64_t n_groups, int64_t capacity) {
  BaPlan p{};
  p.prec = q_dtype != TQ_BF16;
  const int most = ba_groups(p.prec), G = hq / hkv;
  const int64_t rows = n * G, cus = device_cu_count();
  // One group of 16 rows a wave where sequences hold no more on average (a decode step);
  // otherwise as many as the registers take, which share each tile's lookups.
  p.groups = rows <= 16 * std::max<int64_t>(B, 1) ? 1 : most;
  // Prompts whose rows alone fill the card go to the row kernel: nothing to merge.
  p.rows = n_groups == 0 && p.groups > 1 && rows / (16 * most * kBaWaves) * hkv >= cus;
  const int R = 16 * p.groups * (p.rows ? kBaWaves : 1);
  p.items = rows / R + B + 1;
  const int64_t tiles = capacity / 64 + 1;
  auto split_grid = [&](int64_t items) {
    const int64_t pieces = (items * hkv * tiles + kBaWaves - 1) / kBaWaves;
    return (unsigned)std::max<int64_t>(1, std::min(cus, pieces));
  };
  p.grid = p.rows ? (unsigned)std::min<int64_t>(p.items * hkv, UINT_MAX) : split_grid(p.items);
  size_t at = 0;
  auto take = [&](size_t bytes) {
    const size_t here = at;
    at += align_up(bytes, 256);
    return here;
  };
  if (!p.rows) {
    take(kBaHeadBytes);
    take(p.items * sizeof(BaItem));
    p.slots = (size_t)p.grid * 2 * ba_slot_floats(16 * p.groups) * 4;
    take(p.slots);
  }
  if (n_groups > 0) {
    p.pgroups = rows <= 16 * n_groups ? 1 : most;
    p.pitems = rows / (16 * p.pgroups) + n_groups;
    p.pgrid = split_grid(p.pitems);
    p.pslots = (size_t)p.pgrid * 2 * ba_slot_floats(16 * p.pgroups) * 4;
    p.row_bytes = (size_t)n * hq * 66 * 4;
    take(kBaHeadBytes);
    take(p.pitems * sizeof(BaItem));
    take((size_t)n_groups * 4);
    take(p.pslots);
    take(p.row_bytes);
    take(p.row_bytes);
  }
  p.total = at;
  return p;
}

void ba_run(int vbits, const BaArgs& a, bool sub, bool prec, bool rows, int groups, unsigned grid, hipStream_t st) {
  if (vbits == 2) ba_launch<2>(a, sub, prec, rows, groups, grid, st);
  else if (vbits == 3) ba_launch<3>(a, sub, prec, rows, groups, grid, st);
  else ba_launch<4>(a, sub, prec, rows, groups, grid, st);
}

}  // namespace
}  // namespace tq

using namespace tq;

extern "C" {

size_t tq_attention_batch_workspace_bytes(tq_dtype q_dtype, int32_t n_tokens, int32_t hq, int32_t hkv,
                                          int32_t n_seqs, int32_t n_groups, int64_t capacity) {
  if (n_tokens <= 0 || hkv < 1 || hq < hkv || hq % hkv || n_seqs < 0 || n_groups < 0 || capacity < 0) return 0;
  return ba_plan(q_dtype, n_tokens, hq, hkv, n_seqs, n_groups, capacity).total;
}

int tq_attention_batch_paged_dl(const void* q, tq_dtype q_dtype, int32_t n_tokens, int64_t q_stride, int32_t hq,
                                int32_t hkv, int32_t d, const uint8_t* kpairs_pool, const float* knorm_pool,
                                const uint8_t* vtile_pool, const float* vnorm_pool, int64_t num_blocks,
                                int32_t block_size, int32_t vbits, const int32_t* block_tables,
                                int64_t table_stride, int32_t max_blocks, const int32_t* query_start_loc,
                                const int32_t* seq_lens, int32_t n_seqs, const int32_t* group_start_loc,
                                const int32_t* shared_lens, int32_t n_groups, const float* kcentroids,
                                const float* vcentroids, const float* krotation, const float* vrotation,
                                float scale, const tq_score_variant* variant, void* out, int64_t out_stride,
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
  TQ_REQUIRE(p.items * hkv * (p.groups) <= INT_MAX && p.pitems * hkv * 3 <= INT_MAX, "too many query rows in one call");
  TQ_REQUIRE(p.total == 0 || (workspace && workspace_bytes >= p.total), "workspace too small: need %zu bytes", p.total);
  TQ_REQUIRE((reinterpret_cast<uintptr_t>(workspace) & 15u) == 0, "workspace must be 16-byte aligned");

  BaArgs a{};
  a.q = q; a.q_stride = q_stride; a.q_dt = (int)q_dtype;
  a.n_tokens = n_tokens; a.hq = hq; a.hkv = hkv; a.G = hq / hkv; a.B = n_seqs;
  a.query_start = query_start_loc; a.seq_lens = seq_lens;
  a.group_start = n_groups ? group_start_loc : nullptr; a.shared = shared_lens; a.n_groups = n_groups;
  a.kpairs = kpairs_pool; a.knorms = knorm_pool; a.vtiles = vtile_pool; a.vnorms = vnorm_pool;
  a.block_tables = block_tables; a.table_stride = table_stride;
  a.max_blocks = max_blocks; a.bs_log2 = bsl; a.num_blocks = (uint32_t)num_blocks;
  a.cap = empty ? 0 : (int)cap;
  a.kcen = kcentroids; a.vcen = vcentroids; a.krot = krotation; a.vrot = vrotation;
  a.qscale = scale * 1.4426950408889634f;
  if (v.softcap > 0.f) {
    a.cap2 = v.softcap * 1.4426950408889634f;
    a.cap2_inv = 1.f / a.cap2;
  }
  a.slopes = v.alibi_slopes; a.window = v.window; a.prefix_lens = v.prefix_lens; a.token_starts = v.token_starts;
  a.out = out; a.out_stride = out_stride; a.lse = lse; a.zero_tail = zero_tail;
  hipStream_t st = as_stream(stream);
  char* at = static_cast<char*>(workspace);
  auto take = [&](size_t bytes) {
    char* here = at;
    at += align_up(bytes, 256);
    return here;
  };
  if (p.rows) {
    ba_run(vbits, a, bsl < 6, p.prec, true, p.groups, p.grid, st);
    TQ_LAUNCH_CHECK("batch_attn_kernel");
    return TQ_OK;
  }
  a.head = reinterpret_cast<BaHead*>(take(kBaHeadBytes));
  a.items = reinterpret_cast<BaItem*>(take(p.items * sizeof(BaItem)));
  a.max_items = (int)p.items;
  a.slots = reinterpret_cast<float*>(take(p.slots));
  BaPrefix pre{};
  if (n_groups > 0) {
    BaArgs b = a;
    b.over_groups = 1;
    b.head = reinterpret_cast<BaHead*>(take(kBaHeadBytes));
    b.items = reinterpret_cast<BaItem*>(take(p.pitems * sizeof(BaItem)));
    b.max_items = (int)p.pitems;
    b.seg_item = reinterpret_cast<int32_t*>(take((size_t)n_groups * 4));
    b.slots = reinterpret_cast<float*>(take(p.pslots));
    float* mine = reinterpret_cast<float*>(take(p.row_bytes));
    float* theirs = reinterpret_cast<float*>(take(p.row_bytes));
    a.row_sums = mine;
    a.row_stats = mine + (size_t)n_tokens * hq * 64;
    b.row_sums = theirs;
    b.row_stats = theirs + (size_t)n_tokens * hq * 64;
    pre = BaPrefix{b.slots, b.head, b.items, b.seg_item, b.row_sums, b.row_stats, b.max_items, 16 * p.pgroups};
    ba_run(vbits, b, bsl < 6, p.prec, false, p.pgroups, p.pgrid, st);
    TQ_LAUNCH_CHECK("batch_attn_kernel");
  }
  ba_run(vbits, a, bsl < 6, p.prec, false, p.groups, p.grid, st);
  TQ_LAUNCH_CHECK("batch_attn_kernel");
  hipLaunchKernelGGL(batch_combine_kernel, dim3((unsigned)(p.items * hkv * p.groups)), dim3(256), 0, st, a, pre,
                     16 * p.groups, n_groups > 0 ? 1 : 0);
  TQ_LAUNCH_CHECK("batch_combine_kernel");
  return TQ_OK;
}

}  // extern "C"
