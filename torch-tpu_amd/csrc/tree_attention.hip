// Attention over the paged cache in bf16 and e4m3, every key seen: the kernels of tree_attention.h, and the join of all of them.
#include "tree_attention.h"

namespace moe {

// ---- joining ------------------------------------------------------------------------------------------------------------
// Row blocks of the tile that began in stretch blockIdx.x and went on in later ones: the parts in the stretches' order.  A row is taken by
// SPLIT groups of D / 4 lanes, each a share of the parts, which meet in LDS.  Rows of no request and of refused ones become 0.
template <int ROWS, int D, int SPLIT, int HEADS>
__global__ __launch_bounds__(256) void attn_join_kernel(const AttnArgs a) {
  constexpr int lanes = D / 4, per_block = 256 / (lanes * SPLIT);
  __shared__ v4f sh_o[256];
  __shared__ float sh_m[256 / lanes], sh_l[256 / lanes];
  const int tid = threadIdx.x, group = tid / lanes, d = 4 * (tid % lanes), split = group % SPLIT;
  if (blockIdx.y == gridDim.y - 1) {
    const auto nothing = [&](int t) {
      for (int i = tid; i < a.Hq * lanes; i += 256) *(v2i *)(a.out + ((size_t)t * a.Hq * lanes + i) * 4) = (v2i){0, 0};
      if (a.lse)
        for (int i = tid; i < a.Hq; i += 256) a.lse[(size_t)t * a.Hq + i] = -INFINITY;
    };
    for (int b = blockIdx.x; b < a.B; b += gridDim.x) {
      const AttnRequest r = attn_request(a, b);
      if (r.prefix < 0)
        for (int j = 0; j < r.n; j++) nothing(r.t0 + j);
    }
    const int first = min(max(a.cu[0], 0), a.T), end = min(max(a.cu[a.B], 0), a.T);
    for (int t = blockIdx.x; t < first; t += gridDim.x) nothing(t);
    for (int t = end + (int)blockIdx.x; t < a.T; t += gridDim.x) nothing(t);
    return;
  }
  const int *rec = a.records + 8 * blockIdx.x;
  const int w1 = rec[0], kh = rec[3], m_tile = rec[4], side = rec[5], w0 = blockIdx.x;
  const AttnRequest r{rec[1], rec[2], 0, 0};
  if (w1 <= w0) return;
  constexpr int blocks = ROWS / per_block;             // of a head
  const int of_head = blockIdx.y / blocks, first_row = blockIdx.y % blocks * per_block;
  const int in_tile = first_row + group / SPLIT, row = m_tile * ROWS + in_tile;
  if (m_tile * ROWS + first_row >= r.n * a.G) return;
  const auto part = [&](int w) { return ((size_t)(2 * w + (w == w0 ? side : 0)) * HEADS + of_head) * ROWS + in_tile; };
  float m = -INFINITY, l = 0.f;
  v4f o = (v4f){0.f, 0.f, 0.f, 0.f};
  if (row < r.n * a.G) {
    for (int first = w0 + split; first <= w1; first += 4 * SPLIT) {      // four parts asked for at a time (eight: slower where there are four)
      float pm[4], pl[4];
      v4f po[4];
#pragma unroll
      for (int i = 0; i < 4; i++) {
        const size_t at = part(min(first + i * SPLIT, w1));
        pm[i] = a.part_ml[at * 2], pl[i] = a.part_ml[at * 2 + 1];
        po[i] = *(const v4f *)(a.part_o + at * D + d);
      }
      const float before = m;
#pragma unroll
      for (int i = 0; i < 4; i++) {
        if (first + i * SPLIT > w1) pm[i] = -INFINITY, pl[i] = 0.f, po[i] = (v4f){0.f, 0.f, 0.f, 0.f};
        m = fmaxf(m, pm[i]);
      }
      const float top = m == -INFINITY ? 0.f : m;      // (nothing seen so far: weights of 0, not of -inf + inf)
      const float f = __builtin_amdgcn_exp2f(before - top);
      l *= f;
      o *= f;
#pragma unroll
      for (int i = 0; i < 4; i++) {
        const float w = __builtin_amdgcn_exp2f(pm[i] - top);
        l += pl[i] * w;
        o += po[i] * w;
      }
    }
  }
  if (SPLIT > 1) {
    sh_o[tid] = o;
    if (d == 0) sh_m[group] = m, sh_l[group] = l;
    __syncthreads();
    if (split) return;
    m = sh_m[group];
#pragma unroll
    for (int i = 1; i < SPLIT; i++) m = fmaxf(m, sh_m[group + i]);
    l = 0.f;
    o = (v4f){0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < SPLIT; i++) {
      const float f = m == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(sh_m[group + i] - m);
      l += sh_l[group + i] * f;
      o += sh_o[tid + i * lanes] * f;
    }
  }
  attn_store<ROWS, D>(a, r, kh * HEADS + of_head, m_tile, in_tile, d, true, 0, o, m, l);
}

void attn_join(const AttnArgs &a, const AttnPlan &plan, int D, hipStream_t st) {
  using std::integral_constant;
  const auto run = [&](auto dim) {
    constexpr int Dc = decltype(dim)::value;
    const auto join = [&](auto rows, auto split, auto heads) {
      constexpr int R = decltype(rows)::value, S = decltype(split)::value, H = decltype(heads)::value;
      attn_join_kernel<R, Dc, S, H><<<dim3(a.groups, R * H * Dc * S / 1024 + 1), 256, 0, st>>>(a);
    };
    constexpr integral_constant<int, 1> one{};
    if (plan.rows == 16 && plan.heads == 1) join(integral_constant<int, 16>(), integral_constant<int, 8>(), one);
    else if (plan.rows == 16) join(integral_constant<int, 16>(), integral_constant<int, 8>(), integral_constant<int, 2>());
    else if (plan.rows == 64) join(integral_constant<int, 64>(), integral_constant<int, 2>(), one);
    else if (plan.rows == 128) join(integral_constant<int, 128>(), one, one);
    else join(integral_constant<int, 256>(), one, one);
  };
  if (D == 64) run(integral_constant<int, 64>());
  else run(integral_constant<int, 128>());
}

}  // namespace moe

extern "C" size_t moe_tree_attention_workspace_bytes(int T, int Hq, int Hkv, int D, int B, int cache_dtype) {
  using namespace moe;
  if (T < 0 || Hq < 1 || Hkv < 1 || Hq % Hkv || D < 1 || B < 0 || cache_dtype < MOE_DTYPE_BF16 || cache_dtype > MOE_DTYPE_FP4) return 0;
  if (cache_dtype == MOE_DTYPE_FP4) return moe_window_attention_workspace_bytes(T, Hq, Hkv, D, B, cache_dtype);
  return attn_workspace(attn_plan(T, Hq, Hkv, B, cache_dtype, false, false, 1ll << 31), D);          // (shorter caches need no more)
}

extern "C" int moe_tree_attention_tile_rows(int T, int Hq, int Hkv, int B, int cache_dtype, int trees, int table_width, int page_size) {
  using namespace moe;
  if (T < 0 || Hq < 1 || Hkv < 1 || Hq % Hkv || B < 0 || B > MOE_MAX_REQUESTS || (cache_dtype != MOE_DTYPE_BF16 && cache_dtype != MOE_DTYPE_FP8) ||
      table_width < 0 || page_size < 1 || page_size > MOE_MAX_PAGE || (page_size & (page_size - 1)))
    return 0;
  return attn_plan(T, Hq, Hkv, B, cache_dtype, false, trees != 0, (int64_t)table_width * page_size).rows;
}

extern "C" int moe_tree_attention(void *stream, const void *q_bf16, int64_t q_stride, int T, int Hq, int Hkv, int D,
                                  const void *k_cache, const void *v_cache, int cache_dtype, int n_blocks, int64_t k_block_stride,
                                  int64_t v_block_stride, int page_size, const int32_t *block_tables, int64_t table_stride,
                                  int table_width, const int32_t *kv_lens, const int32_t *cu_tokens, int B, const int64_t *masks,
                                  float scale, const float *k_scale, const float *v_scale, void *out_bf16, float *lse,
                                  void *workspace, size_t workspace_bytes) {
  using namespace moe;
  if (cache_dtype != MOE_DTYPE_BF16 && cache_dtype != MOE_DTYPE_FP8) return MOE_E_MODE;
  AttnPlan plan;
  AttnArgs a;
  const int rc = attn_arguments(q_bf16, q_stride, T, Hq, Hkv, D, k_cache, v_cache, cache_dtype, n_blocks, k_block_stride, v_block_stride, page_size,
                                block_tables, table_stride, table_width, kv_lens, cu_tokens, B, masks, scale, k_scale, v_scale, 0, 0, 0, 0, false,
                                out_bf16, lse, workspace, workspace_bytes, plan, a);
  if (rc || !plan.rows) return rc;
  hipStream_t st = (hipStream_t)stream;
  const bool fp8 = cache_dtype == MOE_DTYPE_FP8;
  if (D == 64 && fp8) attn_main<64, MOE_DTYPE_FP8, false>(a, plan, st);
  else if (D == 64) attn_main<64, MOE_DTYPE_BF16, false>(a, plan, st);
  else if (fp8) attn_main<128, MOE_DTYPE_FP8, false>(a, plan, st);
  else attn_main<128, MOE_DTYPE_BF16, false>(a, plan, st);
  attn_join(a, plan, D, st);
  return (int)hipGetLastError();
}
