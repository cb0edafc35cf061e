// Attention of new tokens over a paged cache: one token of each request, a tree of drafted ones, or a causal chunk.
//
//   token j of request b sees the cached keys [0, p), p = kv_len - n, and of the n new ones, which the cache holds as
//   well, those that its mask names (no masks: 0 .. j);   o = sum_key softmax(scale q.key) value
//
// One pass over the keys with the running maximum and sum of the softmax, both fp32, as is the output until its one
// rounding.  A token that sees nothing gives 0 and -inf.
#include <math.h>
#include "moe_common.h"
#include "moe_layout.h"
#include "../../include/moe_hip.h"

namespace moe {

struct AttnArgs {
  const uint16_t *q;
  int64_t q_stride;
  int T, Hq, Hkv, D, B, n_blocks, page_log2, table_width;
  const uint8_t *k_cache, *v_cache;
  int64_t k_block_bytes, v_block_bytes, table_stride;
  const int32_t *tables, *kv_lens, *cu;
  const int64_t *masks;
  float scale;
  const float *k_scale, *v_scale;
  uint16_t *out;
  float *lse;
};

// the request whose tokens hold row t: the last one with cu[b] <= t
__device__ __forceinline__ int attn_request(const int32_t *cu, int B, int t) {
  int lo = 0, hi = B - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (cu[mid] <= t) lo = mid;
    else hi = mid - 1;
  }
  return lo;
}

// A workgroup for each token and query head; groups of LPK lanes take keys in turn, 8 elements a lane.
template <int LPK, bool FP8>
__global__ __launch_bounds__(256) void tree_attention_simple_kernel(const AttnArgs a) {
  constexpr int G = 256 / LPK;
  __shared__ float sh_m[G], sh_l[G], sh_o[G][LPK * 8 + 1];
  const int t = blockIdx.x / a.Hq, h = blockIdx.x % a.Hq, kh = h / (a.Hq / a.Hkv);
  const int grp = threadIdx.x / LPK, L = threadIdx.x % LPK, e = 8 * L;
  const bool live = e < a.D;
  const int b = attn_request(a.cu, a.B, t);
  const int t0 = a.cu[b], n = min(a.cu[b + 1], a.T) - t0, j = t - t0;
  const int kv = min(a.kv_lens[b], a.table_width << a.page_log2), prefix = kv - n;
  const bool here = j >= 0 && j < n && prefix >= 0;
  const uint64_t mask = a.masks ? (uint64_t)a.masks[t] : 0;
  const float sc = a.scale * (a.k_scale ? a.k_scale[kh] : 1.f) * 1.4426950408889634f;
  float q[8], o[8], m = -INFINITY, l = 0.f;
  const v4i raw = live ? *(const v4i *)(a.q + (size_t)t * a.q_stride + (size_t)h * a.D + e) : (v4i){0, 0, 0, 0};
#pragma unroll
  for (int i = 0; i < 8; i++) {
    q[i] = bf16_to_f32((uint16_t)((uint32_t)raw[i / 2] >> (16 * (i & 1))));
    o[i] = 0.f;
  }
  const auto load8 = [&](const uint8_t *at, float *v) {
    if (FP8) {
      const v2i r = *(const v2i *)at;
#pragma unroll
      for (int i = 0; i < 2; i++) {
        const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8(r[i], false), hi = __builtin_amdgcn_cvt_pk_f32_fp8(r[i], true);
        v[4 * i] = lo[0], v[4 * i + 1] = lo[1], v[4 * i + 2] = hi[0], v[4 * i + 3] = hi[1];
      }
    } else {
      const v4i r = *(const v4i *)at;
#pragma unroll
      for (int i = 0; i < 8; i++) v[i] = bf16_to_f32((uint16_t)((uint32_t)r[i / 2] >> (16 * (i & 1))));
    }
  };
  if (here)
    for (int key = grp; key < kv; key += G) {
      const int i = key - prefix;
      if (i >= 0 && !(a.masks ? i < 64 && (mask >> i & 1) : i <= j)) continue;
      const int block = min(max(a.tables[(size_t)b * a.table_stride + (key >> a.page_log2)], 0), a.n_blocks - 1);
      const int64_t within = (((int64_t)(key & ((1 << a.page_log2) - 1)) * a.Hkv + kh) * a.D + e) * (FP8 ? 1 : 2);
      float k[8], v[8], s = 0.f;
      if (live) {
        load8(a.k_cache + block * a.k_block_bytes + within, k);
        load8(a.v_cache + block * a.v_block_bytes + within, v);
#pragma unroll
        for (int x = 0; x < 8; x++) s = fmaf(q[x], k[x], s);
      }
#pragma unroll
      for (int d = 1; d < LPK; d <<= 1) s += __shfl_xor(s, d, 64);
      s *= sc;
      const float m2 = fmaxf(m, s), base = m2 == -INFINITY ? 0.f : m2;
      const float f = exp2f(m - base), p = exp2f(s - base);
      m = m2;
      l = l * f + p;
      if (live)
#pragma unroll
        for (int x = 0; x < 8; x++) o[x] = o[x] * f + p * v[x];
    }
  if (L == 0) sh_m[grp] = m, sh_l[grp] = l;
#pragma unroll
  for (int x = 0; x < 8; x++) sh_o[grp][e + x] = o[x];
  __syncthreads();
  float top = -INFINITY;
  for (int i = 0; i < G; i++) top = fmaxf(top, sh_m[i]);
  const float base = top == -INFINITY ? 0.f : top;
  float sum = 0.f;
  for (int i = 0; i < G; i++) sum += sh_l[i] * exp2f(sh_m[i] - base);
  const float vs = a.v_scale ? a.v_scale[kh] : 1.f;
  for (int d = threadIdx.x; d < a.D; d += 256) {
    float r = 0.f;
    for (int i = 0; i < G; i++) {
      const float f = exp2f(sh_m[i] - base);
      if (f != 0.f) r += sh_o[i][d] * f;
    }
    a.out[((size_t)t * a.Hq + h) * a.D + d] = f32_to_bf16(top == -INFINITY && sum == 0.f ? 0.f : r / sum * vs);
  }
  if (a.lse && threadIdx.x == 0) a.lse[(size_t)t * a.Hq + h] = (top == -INFINITY && sum == 0.f) ? -INFINITY : (base + log2f(sum)) * 0.6931471805599453f;
}

}  // namespace moe

extern "C" size_t moe_tree_attention_workspace_bytes(int T, int Hq, int Hkv, int D, int B) {
  if (T < 0 || Hq < 1 || Hkv < 1 || Hq % Hkv || D < 1 || B < 0) return 0;
  return 256;
}

extern "C" int moe_tree_attention(void *stream, const void *q_bf16, int64_t q_stride, int T, int Hq, int Hkv, int D,
                                  const void *k_cache, const void *v_cache, int cache_dtype, int n_blocks, int64_t k_block_stride,
                                  int64_t v_block_stride, int page_size, const int32_t *block_tables, int64_t table_stride,
                                  int table_width, const int32_t *kv_lens, const int32_t *cu_tokens, int B, const int64_t *masks,
                                  float scale, const float *k_scale, const float *v_scale, void *out_bf16, float *lse,
                                  void *workspace, size_t workspace_bytes) {
  using namespace moe;
  if (cache_dtype != MOE_DTYPE_BF16 && cache_dtype != MOE_DTYPE_FP8) return MOE_E_MODE;
  if (T < 0 || B < 0 || B > MOE_MAX_REQUESTS || Hq < 1 || Hkv < 1 || Hq > 4096 || Hq % Hkv || (D != 64 && D != 128)) return MOE_E_SHAPE;
  const int64_t row = (int64_t)Hkv * D;
  if (n_blocks < 0 || page_size < 1 || page_size > MOE_MAX_PAGE || (page_size & (page_size - 1)) || k_block_stride < page_size * row ||
      v_block_stride < page_size * row || table_width < 0 || (B > 1 && table_stride < table_width) || q_stride < (int64_t)Hq * D ||
      (int64_t)table_width * page_size >= (1ll << 31) || (int64_t)T * Hq >= (1ll << 31))
    return MOE_E_SHAPE;
  if (q_stride % 8 || k_block_stride % 16 || v_block_stride % 16) return MOE_E_ALIGN;
  if (T == 0) return MOE_OK;
  if (B == 0 || !q_bf16 || !out_bf16 || !kv_lens || !cu_tokens || !workspace) return MOE_E_NULL;
  if (table_width && n_blocks && (!block_tables || !k_cache || !v_cache)) return MOE_E_NULL;
  for (const void *p : {q_bf16, k_cache, v_cache, (const void *)out_bf16})
    if ((uintptr_t)p % 16) return MOE_E_ALIGN;
  if ((uintptr_t)workspace % 256) return MOE_E_ALIGN;
  if (workspace_bytes < moe_tree_attention_workspace_bytes(T, Hq, Hkv, D, B)) return MOE_E_WORKSPACE;
  const int fp8 = cache_dtype == MOE_DTYPE_FP8, wide = fp8 ? 1 : 2;
  AttnArgs a{(const uint16_t *)q_bf16, q_stride, T, Hq, Hkv, D, B, n_blocks, __builtin_ctz(page_size), n_blocks ? table_width : 0,
             (const uint8_t *)k_cache, (const uint8_t *)v_cache, k_block_stride * wide, v_block_stride * wide, table_stride, block_tables,
             kv_lens, cu_tokens, masks, scale, k_scale, v_scale, (uint16_t *)out_bf16, lse};
  hipStream_t st = (hipStream_t)stream;
  const unsigned grid = (unsigned)((int64_t)T * Hq);
  if (D == 64 && fp8) tree_attention_simple_kernel<8, true><<<grid, 256, 0, st>>>(a);
  else if (D == 64) tree_attention_simple_kernel<8, false><<<grid, 256, 0, st>>>(a);
  else if (fp8) tree_attention_simple_kernel<16, true><<<grid, 256, 0, st>>>(a);
  else tree_attention_simple_kernel<16, false><<<grid, 256, 0, st>>>(a);
  return (int)hipGetLastError();
}
