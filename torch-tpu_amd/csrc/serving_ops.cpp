// Operators of a serving step around the MoE layer in the namespace my_ops: cache_plan, qk_norm_rope, tree_attention,
// token_logprobs (include/moe_hip.h has their definitions).  Plain host C++ on the C ABI, as my_ops.cpp: at decode sizes
// a call's checks and allocations in Python would take longer than its kernel.  Results are allocated here where
// the caller hands none over; the current device's current stream is used; argument errors through TORCH_CHECK.
// Inference only: none of them records a gradient.
#include <ATen/ATen.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/library.h>

#include <optional>
#include <tuple>

#include "../../include/moe_hip.h"

namespace {

using at::Tensor;
using OptTensor = std::optional<Tensor>;

void *current_stream(const Tensor &t) { return (void *)c10::hip::getCurrentHIPStream(t.device().index()).stream(); }
void check_rc(int rc, const char *what) { TORCH_CHECK(rc == 0, what, ": ", moe_hip_strerror(rc), " (code ", rc, ")"); }

// on the GPU and on the device of `like`
void need_gpu(const Tensor &t, const char *name, const Tensor &like) {
  TORCH_CHECK(t.is_cuda(), name, " must be on the GPU");
  TORCH_CHECK(t.device() == like.device(), name, " must be on the device of the other tensors");
}
void need_vector(const Tensor &t, const char *name, at::ScalarType dtype, int64_t size, const Tensor &like) {
  need_gpu(t, name, like);
  TORCH_CHECK(t.scalar_type() == dtype, name, " must be ", dtype, ", got ", t.scalar_type());
  TORCH_CHECK(t.dim() == 1 && t.size(0) == size, name, " must hold ", size, " values, got a tensor of ", t.sizes());
  TORCH_CHECK(t.is_contiguous(), name, " must be contiguous");
}
// a matrix whose rows are contiguous, at any distance from each other
void need_rows(const Tensor &t, const char *name) {
  TORCH_CHECK(t.stride(1) == 1 || t.size(1) <= 1, name, " must have contiguous rows");
}
int64_t row_stride(const Tensor &t) { return t.size(0) > 1 ? t.stride(0) : t.size(1); }
int fits_int(int64_t v, const char *name) {
  TORCH_CHECK(v >= 0 && v < (1ll << 31), name, " is out of range: ", v);
  return (int)v;
}
template <typename T>
T *data_or_null(const OptTensor &t) {
  return t.has_value() ? (T *)t->data_ptr() : nullptr;
}

// Several results in one allocation: at decode sizes half of a call's time was the allocator's (cache_plan: 9.5 us with one
// allocation a result, 6.0 with one in all).  Each piece begins on 64 bytes and is a plain tensor of its own on the common storage.
class Pieces {
 public:
  explicit Pieces(const Tensor &like) : options_(like.options().dtype(at::kByte)) {}
  // -> where the piece will begin
  int64_t add(int64_t values, at::ScalarType dtype) {
    const int64_t at = bytes_;
    bytes_ += (values * (int64_t)c10::elementSize(dtype) + 63) / 64 * 64;
    return at;
  }
  Tensor piece(int64_t at, at::ScalarType dtype, at::IntArrayRef sizes) {
    if (!buffer_.defined()) buffer_ = at::empty({bytes_}, options_);
    Tensor t = at::detail::make_tensor<c10::TensorImpl>(c10::Storage(buffer_.storage()), buffer_.key_set(), c10::scalarTypeToTypeMeta(dtype));
    t.unsafeGetTensorImpl()->set_storage_offset(at / (int64_t)c10::elementSize(dtype));
    t.unsafeGetTensorImpl()->set_sizes_contiguous(sizes);
    return t;
  }

 private:
  c10::TensorOptions options_;
  int64_t bytes_ = 0;
  Tensor buffer_;
};

struct Cache {
  int dtype, n_blocks, page, heads, dim;
  int64_t k_stride, v_stride;
};
// K and V caches [n_blocks, page_size, Hkv, D]: the last three dimensions contiguous, blocks at any distance
Cache cache_of(const Tensor &k, const Tensor &v, const OptTensor &k_scale, const OptTensor &v_scale, const Tensor &like) {
  TORCH_CHECK(k.dim() == 4 && v.dim() == 4, "k_cache and v_cache must be [n_blocks, page_size, heads, head_dim]");
  TORCH_CHECK(k.sizes() == v.sizes() && k.scalar_type() == v.scalar_type(), "k_cache and v_cache must have the same shape and dtype");
  TORCH_CHECK(k.scalar_type() == at::kBFloat16 || k.scalar_type() == at::kFloat8_e4m3fn, "the caches must be bfloat16 or float8_e4m3fn");
  need_gpu(k, "k_cache", like);
  need_gpu(v, "v_cache", like);
  const int64_t row = k.size(1) * k.size(2) * k.size(3);
  for (const Tensor *t : {&k, &v})
    TORCH_CHECK(t->numel() == 0 || t->size(0) == 0 || t->select(0, 0).is_contiguous(), "a block of a cache must be contiguous");
  const bool fp8 = k.scalar_type() == at::kFloat8_e4m3fn;
  TORCH_CHECK(fp8 || (!k_scale && !v_scale), "k_scale and v_scale belong to a float8_e4m3fn cache");
  if (k_scale) need_vector(*k_scale, "k_scale", at::kFloat, k.size(2), like);
  if (v_scale) need_vector(*v_scale, "v_scale", at::kFloat, k.size(2), like);
  return {fp8 ? MOE_DTYPE_FP8 : MOE_DTYPE_BF16, fits_int(k.size(0), "n_blocks"), fits_int(k.size(1), "page_size"),
          fits_int(k.size(2), "heads"), fits_int(k.size(3), "head_dim"), k.size(0) > 1 ? k.stride(0) : row, v.size(0) > 1 ? v.stride(0) : row};
}

std::tuple<Tensor, Tensor, Tensor, OptTensor, Tensor, Tensor> cache_plan(const Tensor &block_tables, const Tensor &lens,
                                                                         const Tensor &counts, const Tensor &free_blocks,
                                                                         const Tensor &n_free, int64_t page_size, int64_t max_tokens,
                                                                         const OptTensor &parents) {
  TORCH_CHECK(block_tables.dim() == 2 && block_tables.scalar_type() == at::kInt, "block_tables must be [requests, pages] int32");
  need_gpu(block_tables, "block_tables", block_tables);
  need_rows(block_tables, "block_tables");
  const int64_t B = block_tables.size(0);
  need_vector(lens, "lens", at::kInt, B, block_tables);
  need_vector(counts, "counts", at::kInt, B, block_tables);
  TORCH_CHECK(free_blocks.dim() == 1, "free_blocks must be one-dimensional");
  need_vector(free_blocks, "free_blocks", at::kInt, free_blocks.size(0), block_tables);
  need_vector(n_free, "n_free", at::kInt, 1, block_tables);
  const int T = fits_int(max_tokens, "max_tokens");
  if (parents) need_vector(*parents, "parents", at::kInt, T, block_tables);
  c10::DeviceGuard guard(block_tables.device());
  Pieces all(block_tables);
  const int64_t at_cu = all.add(B + 1, at::kInt), at_positions = all.add(T, at::kInt), at_slots = all.add(T, at::kLong),
                at_masks = all.add(parents ? T : 0, at::kLong), at_lens = all.add(B, at::kInt), at_left = all.add(1, at::kInt);
  const Tensor cu = all.piece(at_cu, at::kInt, {B + 1}), positions = all.piece(at_positions, at::kInt, {T}),
               slots = all.piece(at_slots, at::kLong, {T}), kv_lens = all.piece(at_lens, at::kInt, {B}), left = all.piece(at_left, at::kInt, {1});
  OptTensor masks;
  if (parents) masks = all.piece(at_masks, at::kLong, {T});
  check_rc(moe_cache_plan(current_stream(block_tables), (int32_t *)block_tables.data_ptr(), row_stride(block_tables), fits_int(B, "requests"),
                          fits_int(block_tables.size(1), "table width"), lens.data_ptr<int32_t>(), counts.data_ptr<int32_t>(),
                          free_blocks.data_ptr<int32_t>(), fits_int(free_blocks.size(0), "free_blocks"), n_free.data_ptr<int32_t>(),
                          fits_int(page_size, "page_size"), data_or_null<int32_t>(parents), T, cu.data_ptr<int32_t>(),
                          positions.data_ptr<int32_t>(), slots.data_ptr<int64_t>(), data_or_null<int64_t>(masks),
                          kv_lens.data_ptr<int32_t>(), left.data_ptr<int32_t>()),
           "cache_plan");
  return {cu, positions, slots, masks, kv_lens, left};
}

std::tuple<Tensor, OptTensor> qk_norm_rope(const Tensor &qkv, const Tensor &positions, const Tensor &cos_sin, int64_t n_heads,
                                           int64_t n_kv_heads, const OptTensor &q_weight, const OptTensor &k_weight, double eps,
                                           bool interleaved, const OptTensor &k_cache, const OptTensor &v_cache,
                                           const OptTensor &slots, const OptTensor &k_scale, const OptTensor &v_scale,
                                           const OptTensor &out) {
  TORCH_CHECK(qkv.dim() == 2 && qkv.scalar_type() == at::kBFloat16, "qkv must be [tokens, (n_heads + 2 n_kv_heads) head_dim] bfloat16");
  need_gpu(qkv, "qkv", qkv);
  need_rows(qkv, "qkv");
  const int64_t T = qkv.size(0), width = qkv.size(1);
  TORCH_CHECK(n_heads > 0 && n_kv_heads > 0 && n_heads < (1 << 20) && n_kv_heads < (1 << 20) && width % (n_heads + 2 * n_kv_heads) == 0 && width > 0,
              "qkv's width ", width, " must be a multiple of n_heads + 2 n_kv_heads");
  const int64_t D = width / (n_heads + 2 * n_kv_heads);
  need_vector(positions, "positions", at::kInt, T, qkv);
  TORCH_CHECK(cos_sin.dim() == 2 && cos_sin.scalar_type() == at::kFloat && cos_sin.is_contiguous(),
              "cos_sin must be a contiguous [positions, rotated dimensions] float32 tensor");
  need_gpu(cos_sin, "cos_sin", qkv);
  int wt = MOE_DTYPE_BF16;
  for (const auto &[w, name] : {std::pair<const OptTensor &, const char *>(q_weight, "q_weight"), {k_weight, "k_weight"}})
    if (w) {
      TORCH_CHECK(w->scalar_type() == at::kBFloat16 || w->scalar_type() == at::kFloat, name, " must be bfloat16 or float32");
      need_vector(*w, name, w->scalar_type(), D, qkv);
      wt = w->scalar_type() == at::kFloat ? MOE_DTYPE_F32 : MOE_DTYPE_BF16;
    }
  TORCH_CHECK(!q_weight || !k_weight || q_weight->scalar_type() == k_weight->scalar_type(), "q_weight and k_weight must have the same dtype");
  TORCH_CHECK(k_cache.has_value() == v_cache.has_value() && k_cache.has_value() == slots.has_value(),
              "k_cache, v_cache and slots belong together");
  Cache c{MOE_DTYPE_BF16, 0, 1, (int)n_kv_heads, (int)D, n_kv_heads * D, n_kv_heads * D};
  if (k_cache) {
    c = cache_of(*k_cache, *v_cache, k_scale, v_scale, qkv);
    TORCH_CHECK(c.heads == n_kv_heads && c.dim == D, "the caches must hold ", n_kv_heads, " heads of ", D);
    need_vector(*slots, "slots", at::kLong, T, qkv);
  } else {
    TORCH_CHECK(!k_scale && !v_scale, "k_scale and v_scale belong to a float8_e4m3fn cache");
  }
  c10::DeviceGuard guard(qkv.device());
  Tensor q;
  if (out) {
    need_gpu(*out, "out", qkv);
    TORCH_CHECK(out->scalar_type() == at::kBFloat16 && out->is_contiguous() && out->sizes() == at::IntArrayRef({T, n_heads, D}),
                "out must be a contiguous [tokens, n_heads, head_dim] bfloat16 tensor");
    q = *out;
  } else {
    q = at::empty({T, n_heads, D}, qkv.options());
  }
  OptTensor k;
  if (!k_cache) k = at::empty({T, n_kv_heads, D}, qkv.options());
  check_rc(moe_qk_norm_rope(current_stream(qkv), qkv.data_ptr(), row_stride(qkv), fits_int(T, "tokens"), (int)n_heads, (int)n_kv_heads,
                            fits_int(D, "head_dim"), positions.data_ptr<int32_t>(), cos_sin.data_ptr<float>(),
                            fits_int(cos_sin.size(0), "positions"), fits_int(cos_sin.size(1), "rotated dimensions"), interleaved,
                            data_or_null<void>(q_weight), data_or_null<void>(k_weight), wt, (float)eps, q.data_ptr(),
                            data_or_null<void>(k), data_or_null<void>(k_cache), data_or_null<void>(v_cache), c.dtype, c.n_blocks,
                            c.k_stride, c.v_stride, c.page, data_or_null<int64_t>(slots), data_or_null<float>(k_scale),
                            data_or_null<float>(v_scale)),
           "qk_norm_rope");
  return {q, k};
}

std::tuple<Tensor, OptTensor> tree_attention(const Tensor &q, const Tensor &k_cache, const Tensor &v_cache, const Tensor &block_tables,
                                             const Tensor &kv_lens, const Tensor &cu_tokens, const OptTensor &masks,
                                             std::optional<double> scale, const OptTensor &k_scale, const OptTensor &v_scale,
                                             const OptTensor &out, bool return_lse) {
  TORCH_CHECK(q.dim() == 3 && q.scalar_type() == at::kBFloat16, "q must be [tokens, heads, head_dim] bfloat16");
  need_gpu(q, "q", q);
  const int64_t T = q.size(0), Hq = q.size(1), D = q.size(2);
  TORCH_CHECK(T == 0 || q.select(0, 0).is_contiguous(), "a token's heads must be contiguous in q");
  const Cache c = cache_of(k_cache, v_cache, k_scale, v_scale, q);
  TORCH_CHECK(c.dim == D && c.heads > 0 && Hq % c.heads == 0, "q's heads must be a multiple of the cache's ", c.heads, " heads of ", c.dim);
  TORCH_CHECK(block_tables.dim() == 2 && block_tables.scalar_type() == at::kInt, "block_tables must be [requests, pages] int32");
  need_gpu(block_tables, "block_tables", q);
  need_rows(block_tables, "block_tables");
  const int64_t B = block_tables.size(0);
  need_vector(kv_lens, "kv_lens", at::kInt, B, q);
  need_vector(cu_tokens, "cu_tokens", at::kInt, B + 1, q);
  if (masks) need_vector(*masks, "masks", at::kLong, T, q);
  c10::DeviceGuard guard(q.device());
  Tensor o;
  if (out) {
    need_gpu(*out, "out", q);
    TORCH_CHECK(out->scalar_type() == at::kBFloat16 && out->is_contiguous() && out->sizes() == q.sizes(),
                "out must be a contiguous bfloat16 tensor of q's shape");
    o = *out;
  } else {
    o = at::empty({T, Hq, D}, q.options());
  }
  OptTensor lse;
  if (return_lse) lse = at::empty({T, Hq}, q.options().dtype(at::kFloat));
  const int t = fits_int(T, "tokens"), h = fits_int(Hq, "heads"), b = fits_int(B, "requests");
  const size_t need = moe_tree_attention_workspace_bytes(t, h, c.heads, c.dim, b, c.dtype);
  const Tensor ws = at::empty({(int64_t)need}, q.options().dtype(at::kByte));
  check_rc(moe_tree_attention(current_stream(q), q.data_ptr(), T > 1 ? q.stride(0) : Hq * D, t, h, c.heads, c.dim, k_cache.data_ptr(),
                              v_cache.data_ptr(), c.dtype, c.n_blocks, c.k_stride, c.v_stride, c.page, block_tables.data_ptr<int32_t>(),
                              row_stride(block_tables), fits_int(block_tables.size(1), "table width"), kv_lens.data_ptr<int32_t>(),
                              cu_tokens.data_ptr<int32_t>(), b, data_or_null<int64_t>(masks), (float)scale.value_or(1.0 / std::sqrt((double)D)),
                              data_or_null<float>(k_scale), data_or_null<float>(v_scale), o.data_ptr(), data_or_null<float>(lse),
                              ws.data_ptr(), need),
           "tree_attention");
  return {o, lse};
}

std::tuple<Tensor, Tensor, Tensor, Tensor> token_logprobs(const Tensor &logits, const Tensor &tokens, int64_t top_k, double temperature) {
  TORCH_CHECK(logits.dim() == 2, "logits must be [tokens, vocabulary]");
  TORCH_CHECK(logits.scalar_type() == at::kFloat || logits.scalar_type() == at::kBFloat16, "logits must be float32 or bfloat16");
  need_gpu(logits, "logits", logits);
  need_rows(logits, "logits");
  const int64_t T = logits.size(0), V = logits.size(1);
  need_vector(tokens, "tokens", at::kLong, T, logits);
  TORCH_CHECK(top_k >= 0 && top_k <= MOE_MAX_TOPK && top_k <= V, "top_k must be from 0 to ", MOE_MAX_TOPK, " and at most the vocabulary");
  TORCH_CHECK(temperature > 0, "temperature must be positive");
  c10::DeviceGuard guard(logits.device());
  const int dtype = logits.scalar_type() == at::kFloat ? MOE_DTYPE_F32 : MOE_DTYPE_BF16;
  const int t = fits_int(T, "tokens"), v = fits_int(V, "vocabulary");
  const size_t need = moe_token_logprobs_workspace_bytes(t, v, (int)top_k, dtype);
  Pieces all(logits);
  const int64_t at_lp = all.add(T, at::kFloat), at_entropy = all.add(T, at::kFloat), at_top = all.add(T * top_k, at::kFloat), at_ids = all.add(T * top_k, at::kInt);
  const Tensor lp = all.piece(at_lp, at::kFloat, {T}), entropy = all.piece(at_entropy, at::kFloat, {T}),
               top = all.piece(at_top, at::kFloat, {T, top_k}), ids = all.piece(at_ids, at::kInt, {T, top_k});
  const Tensor ws = at::empty({(int64_t)need}, logits.options().dtype(at::kByte));
  check_rc(moe_token_logprobs(current_stream(logits), logits.data_ptr(), dtype, row_stride(logits), t, v, tokens.data_ptr<int64_t>(),
                              (int)top_k, (float)temperature, lp.data_ptr<float>(), entropy.data_ptr<float>(), top.data_ptr<float>(),
                              ids.data_ptr<int32_t>(), ws.data_ptr(), need),
           "token_logprobs");
  return {lp, entropy, top, ids};
}

}  // namespace

// What a schema says of memory: (a!) is written, a result (a) is that tensor where it is handed over, results with the same letter share an
// allocation.  (A result marked as written, (a!), would drop out of autograd: backward would not warn that there is no gradient.)
TORCH_LIBRARY_FRAGMENT(my_ops, m) {
  m.def("cache_plan(Tensor(a!) block_tables, Tensor lens, Tensor counts, Tensor free_blocks, Tensor n_free, int page_size, "
        "int max_tokens, Tensor? parents=None) -> (Tensor(b), Tensor(b), Tensor(b), Tensor(b)?, Tensor(b), Tensor(b))");
  m.def("qk_norm_rope(Tensor qkv, Tensor positions, Tensor cos_sin, int n_heads, int n_kv_heads, Tensor? q_weight=None, "
        "Tensor? k_weight=None, float eps=1e-6, bool interleaved=False, Tensor(a!)? k_cache=None, Tensor(b!)? v_cache=None, "
        "Tensor? slots=None, Tensor? k_scale=None, Tensor? v_scale=None, Tensor(c!)? out=None) -> (Tensor(c), Tensor?)");
  m.def("tree_attention(Tensor q, Tensor k_cache, Tensor v_cache, Tensor block_tables, Tensor kv_lens, Tensor cu_tokens, "
        "Tensor? masks=None, float? scale=None, Tensor? k_scale=None, Tensor? v_scale=None, Tensor(a!)? out=None, "
        "bool return_lse=False) -> (Tensor(a), Tensor?)");
  m.def("token_logprobs(Tensor logits, Tensor tokens, int top_k=0, float temperature=1.0) -> (Tensor(a), Tensor(a), Tensor(a), Tensor(a))");
}

TORCH_LIBRARY_IMPL(my_ops, CompositeExplicitAutograd, m) {
  m.impl("cache_plan", cache_plan);
  m.impl("qk_norm_rope", qk_norm_rope);
  m.impl("tree_attention", tree_attention);
  m.impl("token_logprobs", token_logprobs);
}
