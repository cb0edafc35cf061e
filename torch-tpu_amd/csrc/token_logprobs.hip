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
// equal.  The first chunk gives a bound: the k-th best of 64 groups' best keys, which at least k keys reach.  What reaches it there
// and later - some k keys a chunk where values come in no order - is collected in LDS and sorted by wavefronts, 64 keys at a time.
// Where values come in rising order more is collected than there is room for: the row is then looked over again, the
// bound raised with every chunk.
// Many rows are bound by bytes and by instructions alike: 2048 rows of 100003 bf16 logits, some masked, with 8 alternatives take
// 93 us, 4.4 TB/s, without alternatives 83, the copy rate.  One row of 131072: 12.9 us, two launches that each wait for memory and for sorts.
#include <math.h>
#include "moe_common.h"
#include "moe_layout.h"
#include "lanes.h"
#include "../../include/moe_hip.h"

namespace moe {

constexpr int kLpThreads = 256, kLpVectors = 4;        // vectors of 16 bytes that a thread holds of a chunk
// keys collected at a time: what k groups of four threads hold of a chunk at the most, beside the k kept from before
constexpr int kLpRoom = MOE_MAX_TOPK * 4 * 8 * kLpVectors + 2 * MOE_MAX_TOPK;
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

// Exponents t = (x - m) c cost one instruction as fma(x, c, -off), off = m c rounded: they are then all off by the same shift, m c - off, which
// an fma gives exactly and which goes out of the sums when m changes and at the end.  Where m c is so large that the shift is not
// small (a low temperature, a mask of the type's lowest value) the difference comes first, and there is no shift.
constexpr float kLpFar = 65536.f;                      // (a shift of 2^-9 at the most)
__device__ __forceinline__ bool lp_near(float m, float c) { return fabsf(m * c) < kLpFar; }
__device__ __forceinline__ float lp_shift(float m, float c) { return lp_near(m, c) ? fmaf(m, c, -(m * c)) : 0.f; }

struct LpShared {
  LpStats stats[kLpThreads / 64];
  uint64_t best[kLpThreads];
  uint64_t keys[kLpRoom];
  uint64_t bound;
  int count;
};

// a step of a sorting network: lanes D apart, the larger value to the lower lane where `down`
template <int D>
__device__ __forceinline__ uint64_t lp_step(uint64_t v, bool down) {
  const uint64_t o = lane_xor<D>(v);
  return (((threadIdx.x & D) == 0) == down) == (v > o) ? v : o;
}
template <int D>
__device__ __forceinline__ uint64_t lp_steps(uint64_t v, bool down) {
  v = lp_step<D>(v, down);
  if constexpr (D > 1) v = lp_steps<D / 2>(v, down);
  return v;
}
// a wavefront's 64 keys, the largest in lane 0
__device__ __forceinline__ uint64_t lp_sort(uint64_t v) {
  v = lp_steps<1>(v, (threadIdx.x & 2) == 0);
  v = lp_steps<2>(v, (threadIdx.x & 4) == 0);
  v = lp_steps<4>(v, (threadIdx.x & 8) == 0);
  v = lp_steps<8>(v, (threadIdx.x & 16) == 0);
  v = lp_steps<16>(v, (threadIdx.x & 32) == 0);
  return lp_steps<32>(v, true);
}
// the 64 largest of two sorted 64, sorted
__device__ __forceinline__ uint64_t lp_merge(uint64_t a, uint64_t b) {
  return lp_steps<32>(max(a, __shfl(b, 63 - (threadIdx.x & 63), 64)), true);
}
// The 64 best of the n keys collected, sorted, in every wavefront (0: none): each sorts its share, then they are merged.
__device__ __forceinline__ uint64_t lp_best64(LpShared &sh, int n) {
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  uint64_t v = 0;
  for (int at = 64 * w; at < n; at += kLpThreads) {
    const uint64_t more = lp_sort(at + lane < n ? sh.keys[at + lane] : 0);
    v = at == 64 * w ? more : lp_merge(v, more);
  }
  __syncthreads();
  sh.best[threadIdx.x] = v;
  __syncthreads();
  v = sh.best[lane];
  for (int i = 1; i < kLpThreads / 64 && 64 * i < n; i++) v = lp_merge(v, sh.best[64 * i + lane]);
  return v;
}

// the sums of the whole workgroup, in every thread
__device__ __forceinline__ LpStats lp_block_stats(LpStats v, LpShared &sh, float c) {
  // first the largest, then everything in terms of it: one exponential a lane
  float m = v.m;
  m = fmaxf(m, lane_xor<1>(m));
  m = fmaxf(m, lane_xor<2>(m));
  m = fmaxf(m, lane_xor<4>(m));
  m = fmaxf(m, lane_xor<8>(m));
  m = fmaxf(m, lane_xor<16>(m));
  m = fmaxf(m, lane_xor<32>(m));
  v = lp_join(v, LpStats{m, 0.f, 0.f}, c);
  v.s += lane_xor<1>(v.s), v.w += lane_xor<1>(v.w);
  v.s += lane_xor<2>(v.s), v.w += lane_xor<2>(v.w);
  v.s += lane_xor<4>(v.s), v.w += lane_xor<4>(v.w);
  v.s += lane_xor<8>(v.s), v.w += lane_xor<8>(v.w);
  v.s += lane_xor<16>(v.s), v.w += lane_xor<16>(v.w);
  v.s += lane_xor<32>(v.s), v.w += lane_xor<32>(v.w);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) sh.stats[threadIdx.x >> 6] = v;
  __syncthreads();
  v = sh.stats[0];
#pragma unroll
  for (int i = 1; i < kLpThreads / 64; i++) v = lp_join(v, sh.stats[i], c);
  return v;
}

// sh.bound = the k-th best of 64 groups' best keys (0: fewer than k groups have one), if that is more than it was
__device__ __forceinline__ void lp_raise_bound(uint64_t best, int k, LpShared &sh) {
  __syncthreads();
  sh.best[threadIdx.x] = best;
  __syncthreads();
  if (threadIdx.x < 64) {
    uint64_t v = sh.best[threadIdx.x];
#pragma unroll
    for (int i = 1; i < kLpThreads / 64; i++) v = max(v, sh.best[64 * i + threadIdx.x]);
    v = lp_sort(v);
    if ((int)threadIdx.x == k - 1 && v > sh.bound) sh.bound = v;
  }
  __syncthreads();
}

// The k best of the keys collected stay, in order.
__device__ __forceinline__ void lp_keep_best(int k, LpShared &sh) {
  __syncthreads();
  const int n = sh.count;
  const uint64_t v = lp_best64(sh, n);
  __syncthreads();
  if ((int)threadIdx.x < k) {
    sh.keys[threadIdx.x] = v;
    if ((int)threadIdx.x == k - 1 && v) sh.bound = v;
  }
  if (threadIdx.x == 0) sh.count = min(n, k);
  __syncthreads();
}

// Adds the keys of a thread that reach the bound to those collected; key(i) is 0 where there is none, worth(i) says cheaply that it may.
template <int N, typename Worth, typename Key>
__device__ __forceinline__ void lp_push(Worth worth, Key key, uint64_t bound, LpShared &sh) {
#pragma unroll
  for (int i = 0; i < N; i++) {
    if (!worth(i)) continue;
    const uint64_t v = key(i);
    if (v && v >= bound) {
      const int at = atomicAdd(&sh.count, 1);
      if (at < kLpRoom) sh.keys[at] = v;
    }
  }
}

// One chunk when the keys may come in rising order: where they do not fit, those before are cut to the best, the bound is raised by the
// chunk's own, and what reaches it then is at most k groups' keys.
template <int N, typename Key>
__device__ __forceinline__ void lp_push_careful(Key key, uint64_t best, int k, LpShared &sh) {
  for (int again = 0; again < 2; again++) {
    __syncthreads();
    const int before = sh.count;
    const uint64_t bound = sh.bound;
    __syncthreads();
    lp_push<N>([](int) { return true; }, key, bound, sh);
    __syncthreads();
    if (sh.count <= kLpRoom) return;
    __syncthreads();
    if (threadIdx.x == 0) sh.count = before;
    lp_keep_best(k, sh);
    lp_raise_bound(best, k, sh);
  }
}

// the row's results from its sums and its best keys, in order in the first wavefront
__device__ __forceinline__ void lp_write(const LpArgs &a, int row, float token_logit, const LpStats v, uint64_t key) {
  const float log_s = logf(v.s);
  const bool none = v.m == -INFINITY && v.s == 0.f;    // no token is possible: log 0, and nothing to be uncertain about
  if (threadIdx.x == 0) {
    a.logprobs[row] = none ? -INFINITY : token_logit == -INFINITY && v.s == v.s ? -INFINITY : (token_logit - v.m) * a.inv_temp - log_s;
    a.entropy[row] = none ? 0.f : log_s - 0.6931471805599453f * (v.w / v.s);
  }
  if ((int)threadIdx.x < a.k) {
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

// a thread's values of a chunk
template <bool BF16>
struct LpChunk {
  static constexpr int E = BF16 ? 8 : 4, N = E * kLpVectors;         // of a vector; in all
  v4i raw[kLpVectors];
  __device__ __forceinline__ static int vector(int c0, int u) { return c0 + u * kLpThreads + (int)threadIdx.x; }
  // the vectors from c0 on that lie in the row and before v1 whole (0 for the others)
  __device__ __forceinline__ void load(const uint8_t *aligned, int c0, int v1, int lead, int V) {
#pragma unroll
    for (int u = 0; u < kLpVectors; u++) {
      const int v = vector(c0, u), e0 = v * E - lead;
      raw[u] = (v4i){0, 0, 0, 0};
      if (v < v1 && e0 >= 0 && e0 + E <= V) raw[u] = *(const v4i *)(aligned + (size_t)v * 16);
    }
  }
  __device__ __forceinline__ void values(const uint8_t *aligned, int c0, int v1, int lead, int V, float (&x)[N]) const {
#pragma unroll
    for (int i = 0; i < N; i++) {
      const uint32_t w = (uint32_t)raw[i / E][BF16 ? i % E / 2 : i % E];
      x[i] = __uint_as_float(BF16 ? (i & 1 ? w & 0xffff0000u : w << 16) : w);
    }
    if (c0 * E - lead >= 0 && c0 + kLpThreads * kLpVectors <= v1 && (c0 + kLpThreads * kLpVectors) * E - lead <= V) return;
#pragma unroll
    for (int u = 0; u < kLpVectors; u++) {             // a chunk at an end of the row or the segment
      const int v = vector(c0, u), e0 = v * E - lead;
      if (v < v1 && e0 >= 0 && e0 + E <= V) continue;
#pragma unroll
      for (int i = 0; i < E; i++) {
        const bool there = v < v1 && e0 + i >= 0 && e0 + i < V;
        x[u * E + i] = !there ? -INFINITY : BF16 ? bf16_to_f32(((const uint16_t *)aligned)[(size_t)v * E + i]) : ((const float *)aligned)[(size_t)v * E + i];
      }
    }
  }
  // value i as a key; 0: not of this row and segment, or no number
  __device__ __forceinline__ static uint64_t key(const float (&x)[N], int i, int c0, int v1, int lead, int V) {
    const int v = vector(c0, i / E), e = v * E - lead + i % E;
    return v < v1 && e >= 0 && e < V && x[i] == x[i] ? lp_key(x[i], (uint32_t)e) : 0;
  }
};

template <bool BF16>
__global__ __launch_bounds__(kLpThreads) void token_logprobs_kernel(const LpArgs a) {
  typedef LpChunk<BF16> Chunk;
  constexpr int E = Chunk::E, N = Chunk::N, kChunk = kLpThreads * kLpVectors;
  __shared__ LpShared sh;
  const int row = blockIdx.x / a.n_seg, seg = blockIdx.x % a.n_seg, tid = threadIdx.x;
  const uint8_t *base = (const uint8_t *)a.logits + (size_t)row * a.row_stride * (16 / E);
  // rows of any alignment: vector v holds the elements v E - lead .. + E - 1, the first and the last vector maybe partly
  const int lead = (int)((uintptr_t)base % 16) / (16 / E);
  const uint8_t *aligned = base - lead * (16 / E);
  const int n_vec = (a.V + lead + E - 1) / E, v0 = seg * a.seg_vectors, v1 = min(v0 + a.seg_vectors, n_vec);
  Chunk chunk;
  chunk.load(aligned, v0, v1, lead, a.V);
  const float token_logit = a.n_seg == 1 && tid == 0 ? lp_token_logit(a, row, BF16) : 0.f;
  if (tid == 0) {
    sh.bound = 0;
    sh.count = 0;
  }
  LpStats st{-INFINITY, 0.f, 0.f};
  float off = 0.f, shift = 0.f;                        // of st.m
  bool far = false;
  uint64_t bound = 0;
  float bound_value = -INFINITY;
  for (int c0 = v0; c0 < v1; c0 += kChunk) {
    float x[N];
    chunk.values(aligned, c0, v1, lead, a.V, x);
    chunk.load(aligned, c0 + kChunk, v1, lead, a.V);   // the next one while this one is worked on
    float most = x[0];
#pragma unroll
    for (int i = 1; i + 1 < N; i += 2) most = fmaxf(fmaxf(most, x[i]), x[i + 1]);
    most = fmaxf(most, x[N - 1]);
    if (most > st.m) {
      const float now = lp_shift(most, a.c), d = st.m == -INFINITY ? -1e4f : fmaxf((st.m - most) * a.c, -1e4f) + (now - shift);
      const float f = __builtin_amdgcn_exp2f(d);
      st.w = f * (st.w + d * st.s);
      st.s *= f;
      st.m = most;
      shift = now;
      off = most * a.c;
      far = !lp_near(most, a.c);
    }
    if (__builtin_expect(__any(far), 0)) {
      const float m = st.m == -INFINITY ? 0.f : st.m;
#pragma unroll
      for (int i = 0; i < N; i++) {
        const float t = fmaf(x[i] - m, a.c, shift), e = __builtin_amdgcn_exp2f(t);
        st.s += e;
        st.w = fmaf(e, fmaxf(t, -1000.f), st.w);       // (0 times -inf where a logit is -inf)
      }
    } else {
      float s2 = 0.f, w2 = 0.f;                        // two sums at a time: each waits for its last addition
#pragma unroll
      for (int i = 0; i < N; i += 2) {
        const float t = fmaf(x[i], a.c, -off), e = __builtin_amdgcn_exp2f(t);
        const float t2 = fmaf(x[i + 1], a.c, -off), e2 = __builtin_amdgcn_exp2f(t2);
        st.s += e;
        s2 += e2;
        st.w = fmaf(e, fmaxf(t, -1000.f), st.w);
        w2 = fmaf(e2, fmaxf(t2, -1000.f), w2);
      }
      st.s += s2;
      st.w += w2;
    }
    if (a.k) {
      if (c0 == v0) {
        int at = N;                                    // the first place of the largest value
#pragma unroll
        for (int i = N - 1; i >= 0; i--) at = x[i] == most ? i : at;
        const int v = Chunk::vector(c0, at / E), e = v * E - lead + at % E;
        lp_raise_bound(at < N && v < v1 && e >= 0 && e < a.V ? lp_key(most, (uint32_t)e) : 0, a.k, sh);
        bound = sh.bound;
        bound_value = bound ? lp_value(bound) : -INFINITY;
      }
      if (most >= bound_value) lp_push<N>([&](int i) { return x[i] >= bound_value; }, [&](int i) { return Chunk::key(x, i, c0, v1, lead, a.V); }, bound, sh);
      // After 3 and 8 chunks what is collected gives a better bound, so that fewer keys come from those that follow.
      const int turn = (c0 - v0) / kChunk;
      if ((turn == 2 || turn == 7) && c0 + 2 * kChunk < v1) {
        __syncthreads();
        if (sh.count <= kLpRoom) {
          lp_keep_best(a.k, sh);
          bound = sh.bound;
          bound_value = bound ? lp_value(bound) : -INFINITY;
        }
      }
    }
  }
  const float unshift = __builtin_amdgcn_exp2f(-shift);
  st.w = unshift * (st.w - shift * st.s);
  st.s *= unshift;
  st = lp_block_stats(st, sh, a.c);                    // (ends behind a barrier)
  uint64_t key = 0;
  if (a.k) {
    __syncthreads();
    if (__builtin_expect(sh.count > kLpRoom, 0)) {     // rising values: once more, with care
      __syncthreads();
      if (tid == 0) sh.count = 0;
      for (int c0 = v0; c0 < v1; c0 += kChunk) {
        float x[N];
        chunk.load(aligned, c0, v1, lead, a.V);
        chunk.values(aligned, c0, v1, lead, a.V, x);
        uint64_t best = 0;
#pragma unroll
        for (int i = 0; i < N; i++) best = max(best, Chunk::key(x, i, c0, v1, lead, a.V));
        lp_push_careful<N>([&](int i) { return Chunk::key(x, i, c0, v1, lead, a.V); }, best, a.k, sh);
      }
      __syncthreads();
    }
    key = lp_best64(sh, sh.count);
  }
  if (a.n_seg == 1) {
    lp_write(a, row, token_logit, st, key);
    return;
  }
  const size_t part = (size_t)row * a.n_seg + seg;
  if (tid == 0) {
    a.part_stats[part * 3] = st.m;
    a.part_stats[part * 3 + 1] = st.s;
    a.part_stats[part * 3 + 2] = st.w;
  }
  if (tid < a.k) a.part_keys[part * a.k + tid] = key;
}

// A row's segments: the sums, and of their sorted keys those that reach the k-th best of the segments' first ones.
__global__ __launch_bounds__(kLpThreads) void token_logprobs_join_kernel(const LpArgs a, int bf16) {
  constexpr int N = kLpSegments * MOE_MAX_TOPK / kLpThreads;
  __shared__ LpShared sh;
  const int row = blockIdx.x, tid = threadIdx.x;
  uint64_t keys[N], first = 0;
#pragma unroll
  for (int i = 0; i < N; i++) {
    const int at = i * kLpThreads + tid;
    keys[i] = at < a.n_seg * a.k ? a.part_keys[(size_t)row * a.n_seg * a.k + at] : 0;
  }
  LpStats st{-INFINITY, 0.f, 0.f};
  if (tid < a.n_seg) {
    const float *p = a.part_stats + ((size_t)row * a.n_seg + tid) * 3;
    st = {p[0], p[1], p[2]};
    if (a.k) first = a.part_keys[((size_t)row * a.n_seg + tid) * a.k];
  }
  const float token_logit = tid == 0 ? lp_token_logit(a, row, bf16) : 0.f;
  if (tid == 0) {
    sh.bound = 0;
    sh.count = 0;
  }
  st = lp_block_stats(st, sh, a.c);
  uint64_t key = 0;
  if (a.k) {
    lp_raise_bound(first, a.k, sh);                    // (every key is of a lane of its own: 64 segments at most)
    lp_push<N>([](int) { return true; }, [&](int i) { return keys[i]; }, sh.bound, sh);
    __syncthreads();
    key = lp_best64(sh, sh.count);
  }
  lp_write(a, row, token_logit, st, key);
}

// Segments of a row: two workgroups to a compute unit while there are fewer rows than units, but none of less than a vector a thread.
// (63 rows of 109632 float32: 16.5 us, 19.3 with half or twice as many, 32 with eight times; 390 rows of 19050 bf16: 15 us in one piece, 19 in
// two, 21 in three; 700 rows of 100003: 49 and 60 us in one and two.)
static int lp_segments(int T, int V, int elements) {
  const int n_vec = (V + 2 * elements - 2) / elements, most = (n_vec + kLpThreads - 1) / kLpThreads;
  const int want = T > 0 && T < 256 ? (512 + T - 1) / T : 1;
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
