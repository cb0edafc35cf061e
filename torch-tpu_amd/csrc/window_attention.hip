// Attention over the paged cache with a window and first tokens that stay visible, and over a cache in 4 bits: the LOCAL kernels of
// tree_attention.h.  They are instances of their own, so that calls without a window over bf16 and e4m3 caches keep their registers and times.
//   64 single tokens, 16384 keys in a window of 1024, bf16     37.2 us, 3.7 TB/s: a workgroup's tile at once, then launch, lengths and a tile's end
//   64 single tokens over up to 8192 keys in 4 bits            55.5 us, 3.2 TB/s: half lines of memory, and the conversions
//   one token over 32767 keys in 4 bits                        18.5 us: a chain of launch, tables, a few units and the join
#include <algorithm>
#include "tree_attention.h"

extern "C" size_t moe_window_attention_workspace_bytes(int T, int Hq, int Hkv, int D, int B, int cache_dtype) {
  using namespace moe;
  if (T < 0 || Hq < 1 || Hkv < 1 || Hq % Hkv || D < 1 || B < 0 || cache_dtype < MOE_DTYPE_BF16 || cache_dtype > MOE_DTYPE_FP4) return 0;
  const auto of = [&](int64_t keys) { return attn_workspace(attn_plan(T, Hq, Hkv, B, cache_dtype, true, false, keys), D); };
  return std::max(of(1ll << 31), of(1));               // (two heads to 256 workgroups or one to 512; what lies between needs no more)
}

static moe::AttnPlan window_plan(int T, int Hq, int Hkv, int B, int cache_dtype, int trees, int table_width, int page_size, int window, int sinks) {
  using namespace moe;
  if (T < 0 || Hq < 1 || Hkv < 1 || Hq % Hkv || B < 0 || B > MOE_MAX_REQUESTS || cache_dtype < MOE_DTYPE_BF16 || cache_dtype > MOE_DTYPE_FP4 ||
      table_width < 0 || page_size < 1 || page_size > MOE_MAX_PAGE || (page_size & (page_size - 1)) || window < 0 || sinks < 0)
    return {};
  return attn_plan(T, Hq, Hkv, B, cache_dtype, true, trees != 0, attn_seen((int64_t)table_width * page_size, window, sinks));
}
extern "C" int moe_window_attention_tile_rows(int T, int Hq, int Hkv, int B, int cache_dtype, int trees, int table_width, int page_size, int window,
                                              int sinks) {
  return window_plan(T, Hq, Hkv, B, cache_dtype, trees, table_width, page_size, window, sinks).rows;
}
extern "C" int moe_window_attention_heads(int T, int Hq, int Hkv, int B, int cache_dtype, int trees, int table_width, int page_size, int window, int sinks) {
  return window_plan(T, Hq, Hkv, B, cache_dtype, trees, table_width, page_size, window, sinks).heads;
}

extern "C" int moe_window_attention(void *stream, const void *q_bf16, int64_t q_stride, int T, int Hq, int Hkv, int D, const void *k_cache,
                                    const void *v_cache, int cache_dtype, int n_blocks, int64_t k_block_stride, int64_t v_block_stride,
                                    int page_size, const int32_t *block_tables, int64_t table_stride, int table_width, const int32_t *kv_lens,
                                    const int32_t *cu_tokens, int B, const int64_t *masks, float scale, const void *k_scale, const void *v_scale,
                                    int64_t k_scale_block_stride, int64_t v_scale_block_stride, int window, int sinks, void *out_bf16, float *lse,
                                    void *workspace, size_t workspace_bytes) {
  using namespace moe;
  if (cache_dtype < MOE_DTYPE_BF16 || cache_dtype > MOE_DTYPE_FP4) return MOE_E_MODE;
  AttnPlan plan;
  AttnArgs a;
  const int rc = attn_arguments(q_bf16, q_stride, T, Hq, Hkv, D, k_cache, v_cache, cache_dtype, n_blocks, k_block_stride, v_block_stride, page_size,
                                block_tables, table_stride, table_width, kv_lens, cu_tokens, B, masks, scale, k_scale, v_scale, k_scale_block_stride,
                                v_scale_block_stride, window, sinks, true, out_bf16, lse, workspace, workspace_bytes, plan, a);
  if (rc || !plan.rows) return rc;
  hipStream_t st = (hipStream_t)stream;
  if (cache_dtype == MOE_DTYPE_BF16) D == 64 ? attn_main<64, MOE_DTYPE_BF16, true>(a, plan, st) : attn_main<128, MOE_DTYPE_BF16, true>(a, plan, st);
  else if (cache_dtype == MOE_DTYPE_FP8) D == 64 ? attn_main<64, MOE_DTYPE_FP8, true>(a, plan, st) : attn_main<128, MOE_DTYPE_FP8, true>(a, plan, st);
  else D == 64 ? attn_main<64, MOE_DTYPE_FP4, true>(a, plan, st) : attn_main<128, MOE_DTYPE_FP4, true>(a, plan, st);
  attn_join(a, plan, D, st);
  return (int)hipGetLastError();
}
