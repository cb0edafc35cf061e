// What stands between two blocks of a decoder, in one pass over its rows:
//
//   u = x                                            the block's output
//   u = u rsqrt(mean(u^2) + eps) post_weight         (with a post_weight)
//   h = residual + scale gate u                      the residual stream
//   y = h rsqrt(mean(h^2) + eps) weight              the next block's input
//
// Bound by bytes: every value is read once and written once, so a row stays in the registers of the wavefronts that share it, sums of
// squares are added over lanes by data-parallel moves and over wavefronts in LDS, and y is formed from the h in registers, before
// its rounding.  All of it in fp32 with one rounding to each output.
// 16384 rows of 7168 bf16 values with both norms and a gate per column: 185 to 189 us, 5.0 TB/s, where a large copy reaches 4.85; 9808 rows of 1999
// values, which begin anywhere, with both norms 38 us, 4.1 TB/s, of 2000 32; one row of 7168: 2.9 us, the chain of row, sum over the wavefronts and store.
#include <type_traits>
#include "moe_common.h"
#include "lanes.h"
#include "rows_clash.h"
#include "../../include/moe_hip.h"

namespace moe {

struct NormArgs {
  const uint16_t *x;
  int64_t x_stride;
  const void *residual;
  int64_t residual_stride;
  const void *weight, *post_weight, *gate;
  int64_t gate_row, gate_col;          // strides, of which either may be 0: the same for all rows, for all columns
  uint16_t *y;
  void *h;
  int64_t y_stride, h_stride;
  float scale, eps, over_h;            // 1 / H
  int T, H, residual_f32, weight_f32, gate_f32;
};

// Eight neighbouring values of a row from `place` on.  kWhole: on 16 bytes, kAny: on their own size, which the memory path takes in one
// access too, kFew: rows of fewer than eight.  Of kAny a row's last piece of fewer values is loaded as the row's last eight, of which the first `back` are another lane's and
// count as 0 (they may be overwritten already where a row takes its own place), and stored in pieces of 4, 2 and 1.  (9808 rows of 1999 values with one norm: 34 to 38 us,
// 52 with the last piece value by value.)
constexpr int kFew = 0, kAny = 1, kWhole = 2;
typedef v4i __attribute__((aligned(2))) v4i_any;
typedef v2i __attribute__((aligned(2))) v2i_any;
typedef int __attribute__((aligned(2))) int_any;
typedef v4f __attribute__((aligned(4))) v4f_any;
typedef float v2f_any __attribute__((ext_vector_type(2), aligned(4)));
template <int HOW>
__device__ __forceinline__ void norm_load(const void *row, int place, int H, bool f32, float (&v)[8]) {
  if constexpr (HOW == kFew) {
#pragma unroll
    for (int i = 0; i < 8; i++) {
      v[i] = 0.f;
      if (i < H) v[i] = f32 ? ((const float *)row)[i] : bf16_to_f32(((const uint16_t *)row)[i]);
    }
  } else {
    const int back = HOW == kWhole ? 0 : max(place + 8 - H, 0), at = place - back;
    if (f32) {
      const float *p = (const float *)row + at;
      const v4f a = HOW == kWhole ? *(const v4f *)p : *(const v4f_any *)p, b = HOW == kWhole ? *(const v4f *)(p + 4) : *(const v4f_any *)(p + 4);
#pragma unroll
      for (int i = 0; i < 4; i++) v[i] = a[i], v[4 + i] = b[i];
    } else {
      const uint16_t *p = (const uint16_t *)row + at;
      const v4i w = HOW == kWhole ? *(const v4i *)p : *(const v4i_any *)p;
#pragma unroll
      for (int i = 0; i < 4; i++) v[2 * i] = __uint_as_float((uint32_t)w[i] << 16), v[2 * i + 1] = __uint_as_float((uint32_t)w[i] & 0xffff0000u);
    }
    if constexpr (HOW == kAny) {
#pragma unroll
      for (int i = 0; i < 7; i++) v[i] = i < back ? 0.f : v[i];
    }
  }
}
template <int HOW>
__device__ __forceinline__ void norm_store(void *row, int place, int H, bool f32, const float (&v)[8]) {
  const int count = H - place;
  if constexpr (HOW == kFew) {
#pragma unroll
    for (int i = 0; i < 7; i++) {
      if (i >= H) continue;
      if (f32) ((float *)row)[i] = v[i];
      else ((uint16_t *)row)[i] = (uint16_t)pack2_bf16(v[i], 0.f);
    }
  } else if (HOW == kWhole || count >= 8) {
    if (f32) {
      float *p = (float *)row + place;
      const v4f a = {v[0], v[1], v[2], v[3]}, b = {v[4], v[5], v[6], v[7]};
      if (HOW == kWhole) *(v4f *)p = a, *(v4f *)(p + 4) = b;
      else *(v4f_any *)p = a, *(v4f_any *)(p + 4) = b;
    } else {
      uint16_t *p = (uint16_t *)row + place;
      const v4i w = {(int)pack2_bf16(v[0], v[1]), (int)pack2_bf16(v[2], v[3]), (int)pack2_bf16(v[4], v[5]), (int)pack2_bf16(v[6], v[7])};
      if (HOW == kWhole) *(v4i *)p = w;
      else *(v4i_any *)p = w;
    }
  } else {
    const bool four = count & 4, two = count & 2;
    const float v1 = v[1], v2 = v[2], v3 = v[3], v5 = v[5], v6 = v[6], v7 = v[7];
    const float a = four ? v2 : v6, b = four ? v3 : v7, one = four ? (two ? v1 : v3) : two ? v5 : v7;
    if (f32) {
      float *end = (float *)row + H;
      if (four) *(v4f_any *)(end - 4) = (v4f){v[4], v5, v6, v7};
      if (two) *(v2f_any *)(end - (count & 4) - 2) = (v2f_any){a, b};
      if (count & 1) end[-count] = one;
    } else {
      uint16_t *end = (uint16_t *)row + H;
      if (four) *(v2i_any *)(end - 4) = (v2i){(int)pack2_bf16(v[4], v5), (int)pack2_bf16(v6, v7)};
      if (two) *(int_any *)(end - (count & 4) - 2) = (int)pack2_bf16(a, b);
      if (count & 1) end[-count] = (uint16_t)pack2_bf16(one, 0.f);
    }
  }
}
// row t of a tensor of fp32 or bf16
__device__ __forceinline__ const void *norm_row(const void *base, int64_t at, bool f32) { return (const uint8_t *)base + (at << (f32 ? 2 : 1)); }
__device__ __forceinline__ void *norm_row(void *base, int64_t at, bool f32) { return (uint8_t *)base + (at << (f32 ? 2 : 1)); }

// The sum over the WAVES wavefronts of a row; `turn` names the sum, so that a second one needs no barrier of its own.
template <int WAVES>
__device__ __forceinline__ float row_sum(float v, int turn) {
  v = lane_sum<64>(v);
  if constexpr (WAVES > 1) {
    __shared__ float sh[2][WAVES];
    if ((threadIdx.x & 63) == 0) sh[turn][threadIdx.x >> 6] = v;
    __syncthreads();
    v = 0.f;
#pragma unroll
    for (int i = 0; i < WAVES; i++) v += sh[turn][i];
  }
  return v;
}

// A row to WAVES wavefronts, P pieces of 8 values to a lane.  One wavefront a row: four rows to a workgroup.
template <int WAVES, int P, int HOW>
__global__ __launch_bounds__(WAVES > 1 ? 64 * WAVES : 256) void residual_norm_kernel(const NormArgs a) {
  constexpr int ROWS = WAVES > 1 ? 1 : 4, LANES = 64 * WAVES;
  const int64_t t = (int64_t)blockIdx.x * ROWS + (WAVES > 1 ? 0 : threadIdx.x >> 6);
  if (t >= a.T) return;                                // (whole wavefronts, and no barrier where there are several rows)
  const int lane = WAVES > 1 ? threadIdx.x : threadIdx.x & 63;
  // What a row is multiplied with is asked for together with it where a lane has one piece; of more of them weights wait for the first sum, or fewer
  // wavefronts would find room.  (16384 rows of 7168: one piece to each lane of 16 wavefronts 189 us, two of 8 wavefronts 203, with early weights 240.)
  constexpr bool EARLY = P == 1;
  float u[P][8], h[P][8], w[P][8], w2[EARLY ? P : 1][8], g[EARLY ? P : 1][8];
  const auto place = [&](int p) { return (p * LANES + lane) * 8; };
  const auto live = [&](int p) { return place(p) < a.H; };
  const auto weights = [&](const void *from, int p, float (&to)[8]) {
#pragma unroll
    for (int i = 0; i < 8; i++) to[i] = 1.f;
    if (from && live(p)) norm_load<HOW>(from, place(p), a.H, a.weight_f32, to);
  };
  float one = 1.f;                                     // a gate that is the same for the row
  if (a.gate && !a.gate_col) one = a.gate_f32 ? ((const float *)a.gate)[t * a.gate_row] : bf16_to_f32(((const uint16_t *)a.gate)[t * a.gate_row]);
  const auto gates = [&](int p, float (&to)[8]) {
#pragma unroll
    for (int i = 0; i < 8; i++) to[i] = one;
    if (a.gate && a.gate_col && live(p)) norm_load<HOW>(norm_row(a.gate, t * a.gate_row, a.gate_f32), place(p), a.H, a.gate_f32, to);
  };
#pragma unroll
  for (int p = 0; p < P; p++) {
#pragma unroll
    for (int i = 0; i < 8; i++) u[p][i] = h[p][i] = 0.f;
    if (!live(p)) continue;
    norm_load<HOW>(norm_row(a.x, t * a.x_stride, false), place(p), a.H, false, u[p]);
    if (a.residual) norm_load<HOW>(norm_row(a.residual, t * a.residual_stride, a.residual_f32), place(p), a.H, a.residual_f32, h[p]);
  }
  if constexpr (EARLY) {
    if (a.post_weight) weights(a.post_weight, 0, w2[0]);
    weights(a.weight, 0, w[0]);
    gates(0, g[0]);
  }
  if (a.post_weight) {
    float sum = 0.f;
#pragma unroll
    for (int p = 0; p < P; p++)
#pragma unroll
      for (int i = 0; i < 8; i++) sum = fmaf(u[p][i], u[p][i], sum);
    if constexpr (!EARLY) {
#pragma unroll
      for (int p = 0; p < P; p++) weights(a.post_weight, p, w[p]);
    }
    const float r = 1.0f / sqrtf(row_sum<WAVES>(sum, 0) * a.over_h + a.eps);
#pragma unroll
    for (int p = 0; p < P; p++)
#pragma unroll
      for (int i = 0; i < 8; i++) u[p][i] *= r * (EARLY ? w2[EARLY ? p : 0][i] : w[p][i]);
  }
  if (a.gate) {
#pragma unroll
    for (int p = 0; p < P; p++) {
      float (&by)[8] = g[EARLY ? p : 0];
      if (!EARLY) gates(p, by);
#pragma unroll
      for (int i = 0; i < 8; i++) u[p][i] *= by[i];
    }
  }
  float sum = 0.f;
#pragma unroll
  for (int p = 0; p < P; p++) {
    if constexpr (!EARLY) weights(a.weight, p, w[p]);            // (before the wait for the sum)
#pragma unroll
    for (int i = 0; i < 8; i++) {
      h[p][i] = fmaf(a.scale, u[p][i], h[p][i]);
      sum = fmaf(h[p][i], h[p][i], sum);
    }
    if (live(p) && a.h) norm_store<HOW>(norm_row(a.h, t * a.h_stride, a.residual_f32), place(p), a.H, a.residual_f32, h[p]);
  }
  const float r = 1.0f / sqrtf(row_sum<WAVES>(sum, 1) * a.over_h + a.eps);
#pragma unroll
  for (int p = 0; p < P; p++) {
    if (!live(p)) continue;
#pragma unroll
    for (int i = 0; i < 8; i++) h[p][i] *= r * w[p][i];
    norm_store<HOW>(norm_row(a.y, t * a.y_stride, false), place(p), a.H, false, h[p]);
  }
}

}  // namespace moe

extern "C" int moe_residual_norm(void *stream, const void *x_bf16, int64_t x_stride, int T, int H, const void *residual, int residual_dtype,
                                 int64_t residual_stride, const void *weight, const void *post_weight, int weight_dtype, const void *gate,
                                 int gate_dtype, int64_t gate_row_stride, int64_t gate_col_stride, float scale, float eps, void *y_bf16,
                                 int64_t y_stride, void *residual_out, int64_t residual_out_stride) {
  using namespace moe;
  for (const int t : {residual_dtype, weight_dtype, gate_dtype})
    if (t != MOE_DTYPE_F32 && t != MOE_DTYPE_BF16) return MOE_E_MODE;
  if (T < 0 || H < 1 || H > 32768 || x_stride < H || y_stride < H || (residual && residual_stride < H) || (residual_out && residual_out_stride < H) ||
      !(eps >= 0.f))
    return MOE_E_SHAPE;
  const int pieces = (H + 7) / 8;
  int lanes = 64;                                      // of a row
  while (lanes < pieces && lanes < 1024) lanes *= 2;
  if ((T + 3ll) * lanes >> 32) return MOE_E_SHAPE;     // (a launch has fewer than 2^32 threads)
  if (gate && (gate_row_stride < 0 || gate_col_stride < 0 || gate_col_stride > 1 || (gate_row_stride && gate_col_stride && gate_row_stride < H)))
    return MOE_E_SHAPE;
  if (T == 0) return MOE_OK;
  if (!x_bf16 || !y_bf16) return MOE_E_NULL;
  const int64_t rb = residual_dtype == MOE_DTYPE_F32 ? 4 : 2, wb = weight_dtype == MOE_DTYPE_F32 ? 4 : 2, gb = gate_dtype == MOE_DTYPE_F32 ? 4 : 2;
  for (const void *p : {x_bf16, (const void *)y_bf16})
    if ((uintptr_t)p % 2) return MOE_E_ALIGN;
  if ((uintptr_t)residual % rb || (uintptr_t)residual_out % rb || (uintptr_t)weight % wb || (uintptr_t)post_weight % wb || (uintptr_t)gate % gb)
    return MOE_E_ALIGN;
  // What is written lies over nothing that is read, but a row may take the place of the row that it comes from.
  const int64_t xs = 2 * x_stride, ys = 2 * y_stride, rs = rb * residual_stride, hs = rb * residual_out_stride, row = 2ll * H, wide = rb * H;
  const int64_t gs = gb * gate_row_stride, gate_rows = gate_row_stride ? T : 1, gate_row = gb * (gate_col_stride ? H : 1);
  const auto over = [&](const void *p, int64_t stride, int64_t bytes) {
    const auto on = [&](const void *q, int64_t q_stride, int64_t q_bytes, int64_t rows) { return rows_clash(p, stride, bytes, T, q, q_stride, q_bytes, rows); };
    const auto place_of = [&](const void *q, int64_t q_stride, int64_t q_bytes) { return p == q && (T == 1 || stride == q_stride) && bytes == q_bytes; };
    return (!place_of(x_bf16, xs, row) && on(x_bf16, xs, row, T)) || (!place_of(residual, rs, wide) && on(residual, rs, wide, T)) ||
           on(weight, 0, wb * H, 1) || on(post_weight, 0, wb * H, 1) || on(gate, gs, gate_row, gate_rows);
  };
  if (over(y_bf16, ys, row) || (residual_out && (over(residual_out, hs, wide) || rows_clash(residual_out, hs, wide, T, y_bf16, ys, row, T))))
    return MOE_E_MODE;
  NormArgs a{(const uint16_t *)x_bf16, x_stride, residual, residual_stride, weight, post_weight, gate, gate_row_stride, gate_col_stride,
             (uint16_t *)y_bf16, residual_out, y_stride, residual_out_stride, scale, eps, 1.0f / (float)H, T, H,
             residual_dtype == MOE_DTYPE_F32, weight_dtype == MOE_DTYPE_F32, gate_dtype == MOE_DTYPE_F32};
  // Whether every row begins on 16 bytes and has whole pieces of 8 values.
  bool whole = H % 8 == 0 && x_stride % 8 == 0 && y_stride % 8 == 0 && (!residual || residual_stride % 8 == 0) &&
               (!residual_out || residual_out_stride % 8 == 0) && (!gate || !gate_col_stride || gate_row_stride % 8 == 0);
  for (const void *p : {x_bf16, (const void *)y_bf16, residual, (const void *)residual_out, weight, post_weight, gate_col_stride ? gate : nullptr})
    whole = whole && (uintptr_t)p % 16 == 0;
  hipStream_t st = (hipStream_t)stream;
  const unsigned grid = (unsigned)T;
  const auto run = [&](auto how) {
    constexpr int A = decltype(how)::value;
    if (pieces <= 64) residual_norm_kernel<1, 1, A><<<(grid + 3) / 4, 256, 0, st>>>(a);
    else if (pieces <= 128) residual_norm_kernel<2, 1, A><<<grid, 128, 0, st>>>(a);
    else if (pieces <= 256) residual_norm_kernel<4, 1, A><<<grid, 256, 0, st>>>(a);
    else if (pieces <= 512) residual_norm_kernel<8, 1, A><<<grid, 512, 0, st>>>(a);
    else if (pieces <= 1024) residual_norm_kernel<16, 1, A><<<grid, 1024, 0, st>>>(a);
    else if (pieces <= 2048) residual_norm_kernel<16, 2, A><<<grid, 1024, 0, st>>>(a);
    else residual_norm_kernel<16, 4, A><<<grid, 1024, 0, st>>>(a);
  };
  if (whole) run(std::integral_constant<int, kWhole>());
  else if (H >= 8) run(std::integral_constant<int, kAny>());
  else residual_norm_kernel<1, 1, kFew><<<(grid + 3) / 4, 256, 0, st>>>(a);
  return (int)hipGetLastError();
}
