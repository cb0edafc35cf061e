// Log probabilities of given tokens under rows of logits, with the row's entropy and its most likely tokens.
//
//   y = x / temperature,  lse = log sum exp(y),  logprob = y[token] - lse,  entropy = lse - sum p y,  p = exp(y - lse)
//   alternatives: the k largest x, equal ones by the lower index
//
// One pass over the logits.  A workgroup goes through a row, or a segment of one, in chunks that it holds in registers, and
// keeps per thread m = max x, s = sum 2^((x - m) c) and w = sum 2^((x - m) c) (x - m) c with c = log2(e) / temperature, all
// three rescaled when m grows; then entropy = ln 2 (log2 s - w / s).  Few rows are cut into segments, whose results a second
// launch joins.
// For the alternatives a value and its index become one whole number, (value's bits in order, ~index), so that no two are
// equal.  The k-th best of the threads' best keys is a bound that at least k keys reach and that only k threads' keys can
// pass; what passes it is collected in LDS, later chunks add what beats the bound, and the rank of a key at the end is the
// count of larger ones.
#include <math.h>
#include "moe_common.h"
#include "moe_layout.h"
#include "../../include/moe_hip.h"

namespace moe {

constexpr int kLpThreads = 256, kLpVectors = 4;        // vectors of 16 bytes that a thread holds of a chunk
constexpr int kLpRoom = 2048;                          // keys collected at a time
constexpr int kLpSegments = 64;

struct LpArgs {
  const void *logits;
  int64_t row_stride;
  const int64_t *tokens;
  int T, V, k, n_seg, seg_vectors;
  float inv_temp, c;                                   // 1 / temperature; log2(e) / temperature
  float *logprobs, *entropy, *top_logprobs;
  int32_t *top_ids;
  float *part_stats;                                   // [T, n_seg, 3]
  uint64_t *part_keys;                                 // [T, n_seg, k]
};

__device__ __forceinline__ uint64_t lp_key(float x, uint32_t index) {
  const uint32_t u = __float_as_uint(x + 0.0f);        // (-0 and +0 are equal)
  return ((uint64_t)((u >> 31) ? ~u : u | 0x80000000u) << 32) | (uint32_t)~index;
}
__device__ __forceinline__ float lp_value(uint64_t key) {
  const uint32_t o = (uint32_t)(key >> 32);
  return __uint_as_float((o >> 31) ? o & 0x7fffffffu : ~o);
}

struct LpStats {
  float m, s, w;                                       // m = -inf: nothing seen
};
__device__ __forceinline__ LpStats lp_join(const LpStats a, const LpStats b, float c) {
  const float m = fmaxf(a.m, b.m);
  const float base = m == -INFINITY ? 0.f : m;
  // what is -inf off adds nothing: its sums are 0, or NaN where a NaN was seen
  const float da = fmaxf((a.m - base) * c, -1e4f), db = fmaxf((b.m - base) * c, -1e4f);
  const float fa = exp2f(da), fb = exp2f(db);
  return {m, a.s * fa + b.s * fb, fa * (a.w + da * a.s) + fb * (b.w + db * b.s)};
}

struct LpShared {
  LpStats stats[kLpThreads / 64];
  uint64_t best[kLpThreads];
  uint64_t keys[kLpRoom];
  uint64_t bound;
  int count;
};

// the sums of the whole workgroup, in every thread
__device__ __forceinline__ LpStats lp_block_stats(LpStats v, LpShared &sh, float c) {
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const LpStats o{__shfl_xor(v.m, d, 64), __shfl_xor(v.s, d, 64), __shfl_xor(v.w, d, 64)};
    v = lp_join(v, o, c);
  }
  __syncthreads();
  if ((threadIdx.x & 63) == 0) sh.stats[threadIdx.x >> 6] = v;
  __syncthreads();
  v = sh.stats[0];
#pragma unroll
  for (int i = 1; i < kLpThreads / 64; i++) v = lp_join(v, sh.stats[i], c);
  return v;
}

// sh.bound = the k-th largest of the threads' keys (0: none), if that is more than it was
__device__ __forceinline__ void lp_raise_bound(uint64_t best, int k, LpShared &sh) {
  const uint64_t mine = best ? best : threadIdx.x;     // (a key of a value is larger than any thread's number)
  sh.best[threadIdx.x] = mine;
  __syncthreads();
  int larger = 0;
#pragma unroll 8
  for (int i = 0; i < kLpThreads; i++) larger += sh.best[i] > mine;
  if (larger == k - 1 && best > sh.bound) sh.bound = best;
  __syncthreads();
}

// keeps the k best of the keys collected, in order
__device__ __forceinline__ void lp_keep_best(int k, LpShared &sh) {
  __syncthreads();
  const int n = sh.count;
  constexpr int kPer = kLpRoom / kLpThreads;
  uint64_t mine[kPer];
  int rank[kPer];
#pragma unroll
  for (int i = 0; i < kPer; i++) {
    const int at = i * kLpThreads + threadIdx.x;
    mine[i] = at < n ? sh.keys[at] : 0;
    rank[i] = 0;
  }
  for (int j = 0; j < n; j++) {
    const uint64_t other = sh.keys[j];
#pragma unroll
    for (int i = 0; i < kPer; i++) {
      if (i * kLpThreads >= n) break;
      rank[i] += other > mine[i];
    }
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kPer; i++)
    if (mine[i] && rank[i] < k) {
      sh.keys[rank[i]] = mine[i];
      if (rank[i] == k - 1) sh.bound = mine[i];
    }
  if (threadIdx.x == 0) sh.count = min(n, k);
  __syncthreads();
}

// Adds to the collected keys what beats the bound of N keys a thread; key(i) is 0 where there is none, best the largest.
template <int N, typename Key>
__device__ __forceinline__ void lp_collect(Key key, uint64_t best, bool first, int k, LpShared &sh) {
  if (first) lp_raise_bound(best, k, sh);
  for (int again = 0; again < 2; again++) {
    const int before = sh.count;
    const uint64_t bound = sh.bound;
    __syncthreads();
    if (best >= bound && best) {
#pragma unroll
      for (int i = 0; i < N; i++) {
        const uint64_t v = key(i);
        if (v && v >= bound) {
          const int at = atomicAdd(&sh.count, 1);
          if (at < kLpRoom) sh.keys[at] = v;
        }
      }
    }
    __syncthreads();
    const int n = sh.count;
    if (n <= kLpRoom) {
      if (n > kLpRoom - 32 * N) lp_keep_best(k, sh);   // (k threads' keys have to fit beside what is there)
      return;
    }
    // too many: what was there is cut to the best, and the bound raised by this chunk's own
    __syncthreads();
    if (threadIdx.x == 0) sh.count = before;
    lp_keep_best(k, sh);
    lp_raise_bound(best, k, sh);
  }
}

// the row's results from its sums and the keys kept
__device__ __forceinline__ void lp_write(const LpArgs &a, int row, float token_logit, const LpStats v, const LpShared &sh) {
  const float log_s = logf(v.s);
  const bool none = v.m == -INFINITY && v.s == 0.f;    // no token is possible: log 0, and nothing to be uncertain about
  if (threadIdx.x == 0) {
    a.logprobs[row] = none ? -INFINITY : token_logit == -INFINITY && v.s == v.s ? -INFINITY : (token_logit - v.m) * a.inv_temp - log_s;
    a.entropy[row] = none ? 0.f : log_s - 0.6931471805599453f * (v.w / v.s);
  }
  if ((int)threadIdx.x < a.k) {
    const uint64_t key = (int)threadIdx.x < sh.count ? sh.keys[threadIdx.x] : 0;
    const size_t at = (size_t)row * a.k + threadIdx.x;
    a.top_ids[at] = key ? (int32_t)~(uint32_t)key : -1;
    a.top_logprobs[at] = none ? -INFINITY : key ? (lp_value(key) - v.m) * a.inv_temp - log_s : NAN;
  }
}

__device__ __forceinline__ float lp_token_logit(const LpArgs &a, int row, bool bf16) {
  const int64_t token = a.tokens[row];
  if (token < 0 || token >= a.V) return -INFINITY;     // no such token: probability 0
  const size_t at = (size_t)row * a.row_stride + token;
  return bf16 ? bf16_to_f32(((const uint16_t *)a.logits)[at]) : ((const float *)a.logits)[at];
}

template <bool BF16>
__global__ __launch_bounds__(kLpThreads) void token_logprobs_kernel(const LpArgs a) {
  constexpr int E = BF16 ? 8 : 4, N = E * kLpVectors;  // elements of a vector; of a thread's share of a chunk
  __shared__ LpShared sh;
  const int row = blockIdx.x / a.n_seg, seg = blockIdx.x % a.n_seg, tid = threadIdx.x;
  const uint8_t *base = (const uint8_t *)a.logits + (size_t)row * a.row_stride * (16 / E);
  // rows of any alignment: vector v holds the elements v E - lead .. + E - 1, the first and the last vector maybe partly
  const int lead = (int)((uintptr_t)base % 16) / (16 / E);
  const uint8_t *aligned = base - lead * (16 / E);
  const int n_vec = (a.V + lead + E - 1) / E, v0 = seg * a.seg_vectors, v1 = min(v0 + a.seg_vectors, n_vec);
  const float token_logit = a.n_seg == 1 && tid == 0 ? lp_token_logit(a, row, BF16) : 0.f;
  if (tid == 0) {
    sh.bound = 0;
    sh.count = 0;
  }
  __syncthreads();
  LpStats st{-INFINITY, 0.f, 0.f};
  bool first = true;
  for (int c0 = v0; c0 < v1; c0 += kLpThreads * kLpVectors) {
    float x[N];
#pragma unroll
    for (int u = 0; u < kLpVectors; u++) {
      const int v = c0 + u * kLpThreads + tid, e0 = v * E - lead;
      v4i raw = (v4i){0, 0, 0, 0};
      const bool whole = v < v1 && e0 >= 0 && e0 + E <= a.V;
      if (whole) raw = *(const v4i *)(aligned + (size_t)v * 16);
#pragma unroll
      for (int i = 0; i < E; i++) {
        float f;
        if (BF16) f = bf16_to_f32((uint16_t)((uint32_t)raw[i / 2] >> (16 * (i & 1))));
        else f = __uint_as_float((uint32_t)raw[i & 3]);
        x[u * E + i] = whole ? f : -INFINITY;
      }
      if (!whole && v < v1) {
#pragma unroll
        for (int i = 0; i < E; i++)
          if (e0 + i >= 0 && e0 + i < a.V)
            x[u * E + i] = BF16 ? bf16_to_f32(((const uint16_t *)aligned)[(size_t)v * E + i]) : ((const float *)aligned)[(size_t)v * E + i];
      }
    }
    float most = -INFINITY;
#pragma unroll
    for (int i = 0; i < N; i++) most = fmaxf(most, x[i]);
    if (most > st.m) {
      const float d = st.m == -INFINITY ? -1e4f : fmaxf((st.m - most) * a.c, -1e4f), f = exp2f(d);
      st.w = f * (st.w + d * st.s);
      st.s *= f;
      st.m = most;
    }
    // (the difference first: c times a logit of the type's lowest value, as masks use it, would be -inf)
    const float base = st.m == -INFINITY ? 0.f : st.m;
#pragma unroll
    for (int i = 0; i < N; i++) {
      const float t = (x[i] - base) * a.c, e = __builtin_amdgcn_exp2f(t);
      st.s += e;
      st.w = fmaf(e, fmaxf(t, -1000.f), st.w);         // (0 times -inf where a logit is -inf)
    }
    if (a.k) {
      const float bound = sh.bound ? lp_value(sh.bound) : -INFINITY;
      if (__syncthreads_or(first || most >= bound)) {
        const auto key = [&](int i) -> uint64_t {
          const int e = (c0 + (i / E) * kLpThreads + tid) * E - lead + i % E;
          const bool there = c0 + (i / E) * kLpThreads + tid < v1 && e >= 0 && e < a.V && x[i] == x[i];
          return there ? lp_key(x[i], (uint32_t)e) : 0;
        };
        uint64_t best = 0;
#pragma unroll
        for (int i = 0; i < N; i++) best = max(best, key(i));
        lp_collect<N>(key, best, first, a.k, sh);
        first = false;
      }
    }
  }
  st = lp_block_stats(st, sh, a.c);
  if (a.k) lp_keep_best(a.k, sh);
  if (a.n_seg == 1) {
    lp_write(a, row, token_logit, st, sh);
    return;
  }
  const size_t part = (size_t)row * a.n_seg + seg;
  if (tid == 0) {
    a.part_stats[part * 3] = st.m;
    a.part_stats[part * 3 + 1] = st.s;
    a.part_stats[part * 3 + 2] = st.w;
  }
  if (tid < a.k) a.part_keys[part * a.k + tid] = tid < sh.count ? sh.keys[tid] : 0;
}

__global__ __launch_bounds__(kLpThreads) void token_logprobs_join_kernel(const LpArgs a, int bf16) {
  constexpr int N = kLpSegments * MOE_MAX_TOPK / kLpThreads;
  __shared__ LpShared sh;
  const int row = blockIdx.x, tid = threadIdx.x;
  const float token_logit = tid == 0 ? lp_token_logit(a, row, bf16) : 0.f;
  if (tid == 0) {
    sh.bound = 0;
    sh.count = 0;
  }
  __syncthreads();
  LpStats st{-INFINITY, 0.f, 0.f};
  if (tid < a.n_seg) {
    const float *p = a.part_stats + ((size_t)row * a.n_seg + tid) * 3;
    st = {p[0], p[1], p[2]};
  }
  st = lp_block_stats(st, sh, a.c);
  if (a.k) {
    uint64_t keys[N], best = 0;
#pragma unroll
    for (int i = 0; i < N; i++) {
      const int at = i * kLpThreads + tid;
      keys[i] = at < a.n_seg * a.k ? a.part_keys[(size_t)row * a.n_seg * a.k + at] : 0;
      best = max(best, keys[i]);
    }
    lp_collect<N>([&](int i) { return keys[i]; }, best, true, a.k, sh);
    lp_keep_best(a.k, sh);
  }
  lp_write(a, row, token_logit, st, sh);
}

// Segments of a row: enough workgroups for the chip, but none of less than a vector a thread.
static int lp_segments(int T, int V, int elements) {
  const int n_vec = (V + 2 * elements - 2) / elements, most = (n_vec + kLpThreads - 1) / kLpThreads;
  const int want = T > 0 ? (1024 + T - 1) / T : 1;
  const int n = want < most ? want : most;
  return n < 1 ? 1 : n > kLpSegments ? kLpSegments : n;
}

}  // namespace moe

extern "C" size_t moe_token_logprobs_workspace_bytes(int T, int V, int k, int logits_dtype) {
  using namespace moe;
  if (T < 0 || V < 1 || k < 0 || k > MOE_MAX_TOPK || (logits_dtype != MOE_DTYPE_F32 && logits_dtype != MOE_DTYPE_BF16)) return 0;
  const size_t n = lp_segments(T, V, logits_dtype == MOE_DTYPE_BF16 ? 8 : 4);
  return n == 1 ? 256 : align_up((size_t)T * n * 12, 256) + align_up((size_t)T * n * k * 8, 256) + 256;
}

extern "C" int moe_token_logprobs(void *stream, const void *logits, int logits_dtype, int64_t row_stride, int T, int V,
                                  const int64_t *tokens, int k, float temperature, float *logprobs, float *entropy,
                                  float *top_logprobs, int32_t *top_ids, void *workspace, size_t workspace_bytes) {
  using namespace moe;
  if (logits_dtype != MOE_DTYPE_F32 && logits_dtype != MOE_DTYPE_BF16) return MOE_E_MODE;
  if (T < 0 || V < 1 || V > (1 << 28) || k < 0 || k > MOE_MAX_TOPK || k > V || row_stride < V || !(temperature > 0.f) ||
      !(temperature < INFINITY) || !(1.0f / temperature < 1e30f))
    return MOE_E_SHAPE;
  if (T == 0) return MOE_OK;
  if (!logits || !tokens || !logprobs || !entropy || (k && (!top_logprobs || !top_ids))) return MOE_E_NULL;
  const int bf16 = logits_dtype == MOE_DTYPE_BF16, E = bf16 ? 8 : 4, n_seg = lp_segments(T, V, E);
  if ((uintptr_t)logits % (16 / E)) return MOE_E_ALIGN;
  if ((int64_t)T * n_seg > 0x7fffffff) return MOE_E_SHAPE;
  if (n_seg > 1) {
    if (!workspace) return MOE_E_NULL;
    if (workspace_bytes < moe_token_logprobs_workspace_bytes(T, V, k, logits_dtype)) return MOE_E_WORKSPACE;
    if ((uintptr_t)workspace % 256) return MOE_E_ALIGN;
  }
  const int n_vec = (V + 2 * E - 2) / E;
  LpArgs a{logits, row_stride, tokens, T, V, k, n_seg, (n_vec + n_seg - 1) / n_seg, 1.0f / temperature,
           1.4426950408889634f / temperature, logprobs, entropy, top_logprobs, top_ids, (float *)workspace,
           (uint64_t *)((uint8_t *)workspace + align_up((size_t)T * n_seg * 12, 256))};
  hipStream_t st = (hipStream_t)stream;
  if (bf16) token_logprobs_kernel<true><<<T * n_seg, kLpThreads, 0, st>>>(a);
  else token_logprobs_kernel<false><<<T * n_seg, kLpThreads, 0, st>>>(a);
  if (n_seg > 1) token_logprobs_join_kernel<<<T, kLpThreads, 0, st>>>(a, bf16);
  return (int)hipGetLastError();
}
