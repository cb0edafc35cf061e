// Bookkeeping of a paged cache for one step, on the GPU and in one launch: which new pages each request gets, where its new
// tokens' keys and values go, their positions, and which of a tree's drafted tokens each of them sees.
//
//   need_b = pages(len_b + n_b) - pages(len_b), 0 where the tokens do not fit;  upto_b = need_0 + ... + need_b
//   a request is granted its step when its tokens fit its table row and the batch's rows, and upto_b <= the free pages: what
//   requests before it need and bring counts, granted or not
//   its i-th new page is free[n_free - 1 - (upto_b - need_b + i)]
//
// What bounds it is the launch and a chain of dependent reads (lengths -> sums -> free pages -> stores), not bytes, so it
// is one kernel, and nothing passes from one workgroup to another: every workgroup adds up the whole batch's lengths itself
// (16 KB at the most, from L2) and then serves its own requests, one wavefront each, the new tokens across the lanes.  New
// pages are taken from the free list again where a slot needs them, not read back from the table.
// One request 4.2 us, 1024 requests with trees of up to 64 tokens 6.6 us (7.2 from one call to the next: the host's part).
// A tree's masks come from parents by doubling: after step s a token's mask holds its 2^s nearest ancestors.
#include "moe_common.h"
#include "../../include/moe_hip.h"

namespace moe {

constexpr int kPlanThreads = 256, kPlanPer = MOE_MAX_REQUESTS / kPlanThreads;

struct PlanArgs {
  int32_t *tables;
  int64_t table_stride;
  const int32_t *lens, *counts, *free_blocks, *n_free, *parents;
  int B, W, F, page_log2, T;
  int32_t *cu, *positions, *kv_lens, *n_free_out;
  int64_t *slots, *masks;
};

// inclusive sum over the workgroup's threads; totals of its wavefronts pass through `waves`
__device__ __forceinline__ int64_t block_sum_upto(int64_t v, int64_t *waves, int64_t *total) {
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int64_t o = __shfl_up(v, d, 64);
    if (lane >= d) v += o;
  }
  __syncthreads();
  if (lane == 63) waves[w] = v;
  __syncthreads();
  int64_t before = 0, all = 0;
#pragma unroll
  for (int i = 0; i < kPlanThreads / 64; i++) {
    if (i < w) before += waves[i];
    all += waves[i];
  }
  *total = all;
  return v + before;
}

__global__ __launch_bounds__(kPlanThreads) void cache_plan_kernel(const PlanArgs a) {
  extern __shared__ int32_t lds[];
  int32_t *cu = lds, *first = lds + a.B + 1;        // first new page of a request in the free list's order; -1: not granted
  __shared__ int64_t waves[kPlanThreads / 64];
  const int tid = threadIdx.x, per = (a.B + kPlanThreads - 1) / kPlanThreads, b0 = tid * per;
  const int page = 1 << a.page_log2;
  const int64_t room = (int64_t)a.W << a.page_log2;
  const int64_t n_free = min(max(a.n_free[0], 0), a.F);

  int64_t tokens = 0, all;
  int len[kPlanPer], n[kPlanPer];
#pragma unroll
  for (int i = 0; i < kPlanPer; i++) {
    if (i >= per) break;
    const bool there = b0 + i < a.B;
    len[i] = there ? a.lens[b0 + i] : 0;
    n[i] = there ? max(a.counts[b0 + i], 0) : 0;
    tokens += n[i];
  }
  int64_t at = block_sum_upto(tokens, waves, &all) - tokens;
  int64_t pages = 0;
  int need[kPlanPer];
#pragma unroll
  for (int i = 0; i < kPlanPer; i++) {
    if (i >= per) break;
    const bool fits = len[i] >= 0 && (int64_t)len[i] + n[i] <= room && at + n[i] <= a.T && (!a.parents || n[i] <= 64);
    if (b0 + i < a.B) cu[b0 + i] = (int32_t)min(at, (int64_t)a.T);
    at += n[i];
    const int64_t end = (int64_t)len[i] + n[i];
    need[i] = fits ? (int)(((end + page - 1) >> a.page_log2) - (((int64_t)len[i] + page - 1) >> a.page_log2)) : -1;
    pages += max(need[i], 0);
  }
  if (tid == 0) cu[a.B] = (int32_t)min(all, (int64_t)a.T);
  int64_t upto = block_sum_upto(pages, waves, &all) - pages;
  int64_t taken = 0;
#pragma unroll
  for (int i = 0; i < kPlanPer; i++) {
    if (i >= per) break;
    upto += max(need[i], 0);
    const bool granted = need[i] == 0 || (need[i] > 0 && upto <= n_free);
    if (granted && need[i] > 0) taken = upto;
    if (b0 + i < a.B) first[b0 + i] = granted ? (int32_t)min(upto - need[i], n_free) : -1;
  }
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) taken = max(taken, (int64_t)__shfl_xor(taken, d, 64));
  __syncthreads();
  if ((tid & 63) == 0) waves[tid >> 6] = taken;
  __syncthreads();
  if (blockIdx.x == 0) {
    for (int b = tid; b <= a.B; b += kPlanThreads) a.cu[b] = cu[b];
    if (tid == 0) {
      for (int i = 1; i < kPlanThreads / 64; i++) taken = max(taken, waves[i]);
      a.n_free_out[0] = (int32_t)(n_free - taken);
    }
  }

  const int lane = tid & 63;
  const int64_t top = n_free - 1;
  const int stride = gridDim.x * (kPlanThreads / 64);
  for (int b = blockIdx.x * (kPlanThreads / 64) + (tid >> 6); b < a.B; b += stride) {
    const int t0 = cu[b], here = cu[b + 1] - t0, f = first[b];
    const int l = a.lens[b], c = max(a.counts[b], 0);
    const int have = (int)(((int64_t)l + page - 1) >> a.page_log2);
    int32_t *row = a.tables + (size_t)b * a.table_stride;
    if (lane == 0) a.kv_lens[b] = f >= 0 ? l + c : 0;
    if (f >= 0) {
      const int want = (int)(((int64_t)l + c + page - 1) >> a.page_log2);
      for (int p = have + lane; p < want; p += 64) row[p] = a.free_blocks[top - (f + p - have)];
    }
    for (int j0 = 0; j0 < here; j0 += 64) {                  // (one pass for a tree)
      const int j = j0 + lane;
      const bool live = f >= 0 && j < here;
      uint64_t mask = 1ull << lane;
      if (a.parents) {
        int up = live ? a.parents[t0 + j] : -1;
        if (up >= j || up < 0) up = -1;
#pragma unroll
        for (int s = 0; s < 6; s++) {
          const uint64_t m = __shfl(mask, max(up, 0), 64);
          const int u = __shfl(up, max(up, 0), 64);
          if (up >= 0) {
            mask |= m;
            up = u;
          }
        }
      }
      if (j < here) {
        int64_t slot = -1;
        if (live) {
          const int at_page = (l + j) >> a.page_log2;
          const int block = at_page < have ? row[at_page] : a.free_blocks[top - (f + at_page - have)];
          slot = ((int64_t)block << a.page_log2) + ((l + j) & (page - 1));
        }
        a.positions[t0 + j] = live ? l + (a.parents ? __popcll(mask) - 1 : j) : -1;
        a.slots[t0 + j] = slot;
        if (a.parents) a.masks[t0 + j] = live ? (int64_t)mask : 0;
      }
    }
  }
  // rows of the batch that hold no token
  for (int64_t t = cu[a.B] + (int64_t)blockIdx.x * kPlanThreads + tid; t < a.T; t += (int64_t)gridDim.x * kPlanThreads) {
    a.positions[t] = -1;
    a.slots[t] = -1;
    if (a.parents) a.masks[t] = 0;
  }
}

}  // namespace moe

extern "C" int moe_cache_plan(void *stream, int32_t *block_tables, int64_t table_stride, int B, int table_width, const int32_t *lens,
                              const int32_t *counts, const int32_t *free_blocks, int n_free_max, const int32_t *n_free,
                              int page_size, const int32_t *parents, int T, int32_t *cu_tokens, int32_t *positions, int64_t *slots,
                              int64_t *masks, int32_t *kv_lens, int32_t *n_free_out) {
  using namespace moe;
  if (B < 0 || B > MOE_MAX_REQUESTS || table_width < 0 || n_free_max < 0 || T < 0 || page_size < 1 || page_size > MOE_MAX_PAGE ||
      (page_size & (page_size - 1)) || (B > 1 && table_stride < table_width) || (int64_t)table_width * page_size >= (1ll << 31))
    return MOE_E_SHAPE;
  if (!cu_tokens || !n_free || !n_free_out) return MOE_E_NULL;
  if (B && (!lens || !counts || !kv_lens || (table_width && !block_tables))) return MOE_E_NULL;
  if ((n_free_max && !free_blocks) || (T && (!positions || !slots || (parents && !masks)))) return MOE_E_NULL;
  // Every workgroup reads all lengths, the stack and its count while others write already: what is written has to lie apart from what is read.
  struct Range {
    const void *at;
    int64_t bytes;
    bool meets(const Range &o) const {
      return bytes > 0 && o.bytes > 0 && (uintptr_t)at < (uintptr_t)o.at + o.bytes && (uintptr_t)o.at < (uintptr_t)at + bytes;
    }
  };
  const Range read[] = {{lens, 4ll * B}, {counts, 4ll * B}, {free_blocks, 4ll * n_free_max}, {n_free, 4}, {parents, parents ? 4ll * T : 0}};
  const Range written[] = {{cu_tokens, 4ll * (B + 1)}, {positions, 4ll * T}, {slots, 8ll * T}, {masks, parents ? 8ll * T : 0}, {kv_lens, 4ll * B},
                           {n_free_out, 4}};
  const Range table{block_tables, B ? 4 * ((B - 1) * table_stride + table_width) : 0};
  for (const Range &r : read) {
    for (const Range &w : written)
      if (w.meets(r)) return MOE_E_MODE;
    if (table.meets(r))                                // (something may lie between the rows)
      for (int b = 0; b < B; b++)
        if (Range{block_tables + b * table_stride, 4ll * table_width}.meets(r)) return MOE_E_MODE;
  }
  PlanArgs a{block_tables, table_stride, lens, counts, free_blocks, n_free, T ? parents : nullptr, B, table_width, n_free_max,
             __builtin_ctz(page_size), T, cu_tokens, positions, kv_lens, n_free_out, slots, masks};
  const int64_t rows = ((int64_t)B + 3) / 4, fill = ((int64_t)T + 2047) / 2048;
  const int64_t grid = rows > fill ? rows : fill;
  cache_plan_kernel<<<(unsigned)(grid < 1 ? 1 : grid > 1024 ? 1024 : grid), kPlanThreads, (size_t)(2 * B + 1) * 4, (hipStream_t)stream>>>(a);
  return (int)hipGetLastError();
}
