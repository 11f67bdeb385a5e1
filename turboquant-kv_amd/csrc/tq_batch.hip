// tq_batch.hip -- a serving step's batch metadata from device lengths: block tables, slot
// maps and token positions, and the groups of requests that share a prefix, on gfx950.
//
// Nothing here reads lengths on the host, so a step that is captured into a graph replays
// with the lengths its tensors hold then.  No atomics decide an order: the results are the
// same on every run.

#include "tq_common.h"

#include <climits>

namespace tq {
namespace {

constexpr int kPlanThreads = 512;       // tokens of a workgroup (256: 8192 requests 37 us, not 25)
constexpr int kPlanMaxRequests = 8192;  // request starts and first fresh blocks in LDS (64 KB)

// Exclusive sum over the workgroup of one value per thread; `total` gets the whole sum.
template <int THREADS>
__device__ __forceinline__ int64_t block_scan(int64_t v, int64_t* part, int64_t* total) {
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
  int64_t before = 0, all = 0;
#pragma unroll
  for (int w = 0; w < THREADS / 64; ++w) {
    const int64_t p = part[w];
    if (w < wave) before += p;
    all += p;
  }
  *total = all;
  return before + incl - v;
}

// a / b for 0 <= a, 0 < b: positions rarely need 64 bits, whose division takes ten times as long.
__device__ __forceinline__ int64_t plan_div(int64_t a, int b) {
  return (a >> 32) == 0 ? (int64_t)((uint32_t)a / (uint32_t)b) : a / b;
}

struct PlanArgs {
  const int32_t* new_lens;
  const int32_t* context_lens;
  int R;
  int32_t* tables;  // [R][width], rows of stride elements
  int64_t stride;
  int width;
  const int32_t* free_blocks;
  int64_t n_free;
  const int32_t* free_start;  // null: 0
  int bs;
  int n_tokens;
  int32_t* query_start;  // [R + 1]
  int32_t* seq_lens;     // [R]
  int64_t* slots;        // [n_tokens]
  int64_t* positions;    // [n_tokens]
  int32_t* token_request;
  int32_t* blocks_used;  // [1]
};

// Every workgroup scans the requests' lengths itself (R of them from L2, no second launch) and
// then serves a token a thread (four a thread: 9.4 us for 1024 requests of 4 tokens, not 5.5): a
// binary search in the starts names a token's request, and the block of its position is the
// table's (written before the step) or, past the blocks the request held, one of the free
// list.  The token that opens a fresh block stores its id in the table: fresh entries are only
// written here and held ones only read, so workgroups do not wait for each other.  Latency bounds
// it: 3.6 us for 16 requests, 25 for 8192.
__global__ __launch_bounds__(kPlanThreads) void paged_plan_kernel(PlanArgs a) {
  __shared__ int32_t start_s[kPlanMaxRequests + 1];
  __shared__ int32_t first_s[kPlanMaxRequests];
  __shared__ int64_t part[kPlanThreads / 64];
  const int tid = threadIdx.x;
  const int per = (a.R + kPlanThreads - 1) / kPlanThreads;
  const int r0 = min(a.R, tid * per), r1 = min(a.R, r0 + per);
  int64_t sum = 0, all;
  for (int r = r0; r < r1; ++r) sum += max(0, a.new_lens[r]);
  int64_t at = block_scan<kPlanThreads>(sum, part, &all);
  const int live = (int)min<int64_t>(all, a.n_tokens);
  sum = 0;
  for (int r = r0; r < r1; ++r) {
    const int n = max(0, a.new_lens[r]), old = max(0, a.context_lens[r]);
    const int begin = (int)min<int64_t>(at, a.n_tokens), end = (int)min<int64_t>(at + n, a.n_tokens);
    start_s[r] = begin;
    const int64_t len = min<int64_t>((int64_t)old + (end - begin), INT_MAX);
    const int64_t takes = plan_div(len + a.bs - 1, a.bs) - plan_div((int64_t)old + a.bs - 1, a.bs);
    first_s[r] = (int)takes;
    sum += takes;
    if (blockIdx.x == 0) {
      a.query_start[r] = begin;
      a.seq_lens[r] = (int)len;
    }
    at += n;
  }
  int64_t used;
  int64_t before = block_scan<kPlanThreads>(sum, part, &used);
  for (int r = r0; r < r1; ++r) {
    const int takes = first_s[r];
    first_s[r] = (int)before;  // at most one block per new token: fits 32 bits
    before += takes;
  }
  if (tid == 0) {
    start_s[a.R] = live;
    if (blockIdx.x == 0) {
      a.query_start[a.R] = live;
      a.blocks_used[0] = (int)used;
    }
  }
  __syncthreads();

  const int64_t fs = a.free_start ? a.free_start[0] : 0;
  const int64_t i64 = (int64_t)blockIdx.x * kPlanThreads + tid;
  if (i64 >= a.n_tokens) return;
  const int i = (int)i64;
  if (i >= live) {
    a.slots[i] = -1;
    a.positions[i] = 0;
    a.token_request[i] = -1;
    return;
  }
  int lo = 0, hi = a.R;  // the last request that starts at or before i, and so holds it
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (start_s[mid] <= i) lo = mid;
    else hi = mid;
  }
  const int r = lo, old = max(0, a.context_lens[r]);
  const int64_t pos = (int64_t)old + (i - start_s[r]);
  const int64_t j = plan_div(pos, a.bs), held = plan_div((int64_t)old + a.bs - 1, a.bs);
  const int in = (int)(pos - j * a.bs);
  int blk = -1;
  if (j < held) {
    if (j < a.width) blk = a.tables[r * a.stride + j];
  } else {
    const int64_t f = fs + first_s[r] + (j - held);
    if (f >= 0 && f < a.n_free) blk = a.free_blocks[f];
    if (j >= a.width) blk = -1;
    else if (in == 0) a.tables[r * a.stride + j] = blk;
  }
  a.slots[i] = blk < 0 ? -1 : (int64_t)blk * a.bs + in;
  a.positions[i] = pos;
  a.token_request[i] = r;
}

// Tokens of the blocks that the tables of requests r - 1 and r > 0 both begin with, of those
// wholly inside both contexts.  A wave per pair of rows, 256 entries a step, and the next
// step's entries requested before this one's are compared.
__device__ __forceinline__ int common_tokens(const int32_t* __restrict__ tables, int64_t stride, int width,
                                             const int32_t* __restrict__ lens, int r, int bs) {
  const int lane = threadIdx.x & 63;
  const int n = min(width, max(0, min(lens[r - 1], lens[r])) / bs);
  const int32_t* x = tables + (int64_t)(r - 1) * stride;
  const int32_t* y = x + stride;
  int same = n;
  constexpr int kStep = 256;
  int va[4], vb[4];
  auto load = [&](int base, int* p, const int32_t* src) {
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int j = base + 64 * k + lane;
      p[k] = j < n ? src[j] : -1;
    }
  };
  load(0, va, x);
  load(0, vb, y);
  for (int base = 0; base < n; base += kStep) {
    int wa[4], wb[4];
    load(base + kStep, wa, x);
    load(base + kStep, wb, y);
    bool done = false;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int j = base + 64 * k + lane;
      const unsigned long long off = __ballot(j < n && (va[k] != vb[k] || va[k] < 0));
      if (!done && off) {
        same = base + 64 * k + __builtin_ctzll(off);
        done = true;
      }
      va[k] = wa[k];
      vb[k] = wb[k];
    }
    if (done) break;
  }
  return same * bs;
}

__global__ __launch_bounds__(256) void common_blocks_kernel(const int32_t* __restrict__ tables, int64_t stride,
                                                            int width, const int32_t* __restrict__ lens, int R,
                                                            int bs, int32_t* __restrict__ common) {
  const int r = blockIdx.x * 4 + (threadIdx.x >> 6);
  if (r >= R) return;
  const int n = r > 0 ? common_tokens(tables, stride, width, lens, r, bs) : 0;
  if ((threadIdx.x & 63) == 0) common[r] = n;
}

constexpr int kGroupThreads = 1024;

constexpr int kGroupFew = 64;         // requests, and entries of their tables, of a step whose one
constexpr int kGroupEntries = 16384;  // workgroup compares the tables too

// The groups: maximal runs of requests whose neighbours share `least` tokens or more.  One
// workgroup; the run's minimum by atomics in LDS (a minimum does not depend on their order).
// FEW: its waves compare the tables of up to kGroupFew requests themselves (common is null).
template <bool FEW>
__global__ __launch_bounds__(kGroupThreads) void prefix_groups_kernel(const int32_t* __restrict__ tables, int64_t stride,
                                                                      int width, const int32_t* __restrict__ lens,
                                                                      int bs, const int32_t* __restrict__ common, int R,
                                                                      int least, int32_t* __restrict__ starts,
                                                                      int32_t* __restrict__ shared) {
  __shared__ int32_t low[FEW ? kGroupFew : kPlanMaxRequests];
  __shared__ int32_t common_s[FEW ? kGroupFew : 1];
  __shared__ int64_t part[kGroupThreads / 64];
  const int tid = threadIdx.x;
  if constexpr (FEW) {
    for (int r = 1 + (tid >> 6); r < R; r += kGroupThreads / 64) {
      const int n = common_tokens(tables, stride, width, lens, r, bs);
      if ((tid & 63) == 0) common_s[r] = n;
    }
    if (tid == 0) common_s[0] = 0;
    __syncthreads();
    common = common_s;
  }
  for (int r = tid; r < R; r += kGroupThreads) low[r] = INT_MAX;
  const int per = (R + kGroupThreads - 1) / kGroupThreads;
  const int r0 = min(R, tid * per), r1 = min(R, r0 + per);
  int opens = 0;
  for (int r = r0; r < r1; ++r) opens += r == 0 || common[r] < least;
  int64_t n_groups;
  int g = (int)block_scan<kGroupThreads>(opens, part, &n_groups) - 1;  // its barriers order `low`
  for (int r = r0; r < r1; ++r) {
    const int c = common[r];
    if (r == 0 || c < least) starts[++g] = r;
    else atomicMin(&low[g], c);
  }
  __syncthreads();
  for (int r = tid; r < R; r += kGroupThreads) {
    shared[r] = r < n_groups && low[r] != INT_MAX ? low[r] : 0;
    if (r >= n_groups) starts[r] = R;
  }
  if (tid == 0) starts[R] = R;
}

}  // namespace
}  // namespace tq

using namespace tq;

extern "C" {

int tq_paged_batch_plan(const int32_t* new_lens, const int32_t* context_lens, int32_t n_requests,
                        int32_t* block_tables, int64_t table_stride, int32_t max_blocks,
                        const int32_t* free_blocks, int64_t n_free, const int32_t* free_start,
                        int32_t block_size, int32_t n_tokens, int32_t* query_start_loc, int32_t* seq_lens,
                        int64_t* slot_mapping, int64_t* positions, int32_t* token_request,
                        int32_t* blocks_used, void* stream) {
  TQ_REQUIRE(n_requests >= 0 && n_requests <= kPlanMaxRequests, "a plan takes 0-%d requests, got %d",
             kPlanMaxRequests, n_requests);
  TQ_REQUIRE(block_size >= 1, "block_size must be positive, got %d", block_size);
  TQ_REQUIRE(n_tokens >= 0 && max_blocks >= 0 && n_free >= 0, "bad sizes");
  TQ_REQUIRE(table_stride >= max_blocks, "table rows of %d entries overlap at a stride of %lld", max_blocks,
             (long long)table_stride);
  TQ_REQUIRE(query_start_loc && blocks_used && (n_requests == 0 || (new_lens && context_lens && seq_lens)) &&
                 (n_tokens == 0 || (slot_mapping && positions && token_request)) &&
                 (n_requests == 0 || max_blocks == 0 || block_tables) && (n_free == 0 || free_blocks),
             "null pointer argument");
  PlanArgs a{new_lens, context_lens, n_requests, block_tables, table_stride, max_blocks, free_blocks, n_free,
             free_start, block_size, n_tokens, query_start_loc, seq_lens, slot_mapping, positions,
             token_request, blocks_used};
  const unsigned grid = n_tokens ? (unsigned)(((int64_t)n_tokens + kPlanThreads - 1) / kPlanThreads) : 1u;
  hipLaunchKernelGGL(paged_plan_kernel, dim3(grid), dim3(kPlanThreads), 0, as_stream(stream), a);
  TQ_LAUNCH_CHECK("paged_plan_kernel");
  return TQ_OK;
}

size_t tq_shared_prefix_groups_workspace_bytes(int32_t n_requests) {
  return n_requests > 0 ? (size_t)n_requests * 4 : 0;
}

int tq_shared_prefix_groups(const int32_t* block_tables, int64_t table_stride, int32_t max_blocks,
                            const int32_t* context_lens, int32_t n_requests, int32_t block_size,
                            int32_t min_tokens, int32_t* group_start_loc, int32_t* shared_lens,
                            void* workspace, size_t workspace_bytes, void* stream) {
  TQ_REQUIRE(n_requests >= 0 && n_requests <= kPlanMaxRequests, "groups are found among 0-%d requests, got %d",
             kPlanMaxRequests, n_requests);
  TQ_REQUIRE(block_size >= 1, "block_size must be positive, got %d", block_size);
  TQ_REQUIRE(min_tokens >= 1, "min_tokens must be positive, got %d", min_tokens);
  TQ_REQUIRE(max_blocks >= 0 && table_stride >= max_blocks, "table rows of %d entries overlap at a stride of %lld",
             max_blocks, (long long)table_stride);
  TQ_REQUIRE((int64_t)max_blocks * block_size <= INT_MAX, "the tables' capacity exceeds 2^31 tokens");
  TQ_REQUIRE(group_start_loc && (n_requests == 0 || (context_lens && shared_lens && (max_blocks == 0 || block_tables))),
             "null pointer argument");
  const size_t need = tq_shared_prefix_groups_workspace_bytes(n_requests);
  TQ_REQUIRE(need == 0 || (workspace && workspace_bytes >= need), "workspace too small: need %zu bytes", need);
  hipStream_t st = as_stream(stream);
  int32_t* common = static_cast<int32_t*>(workspace);
  // One launch for few requests, whose tables one workgroup compares nearly as fast: 4.8 us for 32
  // rows of 256 entries where two take 2.6 us each and a gap; 10.8 and 9.4 + 2.6 for 4 of 4096.
  const bool few = n_requests <= kGroupFew && (int64_t)n_requests * max_blocks <= kGroupEntries;
  if (few) {
    hipLaunchKernelGGL((prefix_groups_kernel<true>), dim3(1), dim3(kGroupThreads), 0, st, block_tables, table_stride,
                       max_blocks, context_lens, block_size, nullptr, n_requests, min_tokens, group_start_loc, shared_lens);
    TQ_LAUNCH_CHECK("prefix_groups_kernel");
    return TQ_OK;
  }
  if (n_requests > 0) {
    hipLaunchKernelGGL(common_blocks_kernel, dim3((unsigned)(n_requests + 3) / 4), dim3(256), 0, st, block_tables,
                       table_stride, max_blocks, context_lens, n_requests, block_size, common);
    TQ_LAUNCH_CHECK("common_blocks_kernel");
  }
  hipLaunchKernelGGL((prefix_groups_kernel<false>), dim3(1), dim3(kGroupThreads), 0, st, block_tables, table_stride,
                     max_blocks, context_lens, block_size, common, n_requests, min_tokens, group_start_loc, shared_lens);
  TQ_LAUNCH_CHECK("prefix_groups_kernel");
  return TQ_OK;
}

}  // extern "C"
