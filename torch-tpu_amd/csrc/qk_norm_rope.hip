// Norms of queries and keys per head, the position rotation, and the way of keys and values into a paged cache, in one
// pass over the fused projection's rows [q heads | k heads | v heads].
//
//   y = x * rsqrt(mean(x^2) + eps) * w        (heads with a weight; over the D elements of a head, fp32)
//   (y_a, y_b) -> (y_a cos - y_b sin, y_b cos + y_a sin)     pairs (i, i + R/2) or (2i, 2i + 1) of the first R elements
//
// One rounding at the end: to bf16, to e4m3 after the division by the head's scale, or to 4 bits after the division by a power of two
// that 32 neighbouring elements share, the least that leaves them at 7 or below: what lies between 6, the largest code, and 7 is then off by no more than the
// half step of 1 that values above 4 are off by anyway, and a value is never off by more than a fifth of the 32's largest (5, that goes to 4).
// It is bound by bytes, so a value is read once and written once.  A lane holds 8 neighbouring elements of a head, D/8 lanes a head
// (rounded up to a power of two); the sum of squares is taken over those lanes, and the partner of an (i, i + R/2) pair comes
// from the lane R/16 further as the two bf16 that the register holds.  A lane's angles and weights are the same for every head, so it
// takes several heads of a token where there are tokens enough to fill the chip.
// 16384 tokens of 32 + 2 x 4 heads of 128 into an e4m3 cache: 72 us, 4.5 TB/s, where a large copy reaches 4.9; into one in 4 bits 67 us;
// one token: 3.5 us, the chain of position, angles and the sum across lanes.
#include <type_traits>
#include "moe_common.h"
#include "lanes.h"
#include "../../include/moe_hip.h"

namespace moe {

struct RopeArgs {
  const uint16_t *qkv;
  int64_t row_stride;
  const int32_t *positions;
  const float *cos_sin;
  const void *q_weight, *k_weight;
  uint16_t *q_out, *k_out;
  uint8_t *k_cache, *v_cache;
  int64_t k_block_bytes, v_block_bytes, n_slots;
  const int64_t *slots;
  const float *k_scale, *v_scale;
  uint8_t *k_powers, *v_powers;        // of a cache in 4 bits: [n_blocks][page][Hkv][D / 32] exponents
  int64_t k_powers_block, v_powers_block;
  float eps;
  int T, Hq, Hkv, D, R, P, page_log2, weights_bf16, interleaved, cache_fp8, groups_per_token;
};

__device__ __forceinline__ void load_weight(const void *w, int is_bf16, int e, float *out) {
  if (is_bf16) {
    const v4i raw = *(const v4i *)((const uint16_t *)w + e);
#pragma unroll
    for (int i = 0; i < 4; i++) {
      out[2 * i] = bf16_to_f32((uint16_t)((uint32_t)raw[i] & 0xffff));
      out[2 * i + 1] = bf16_to_f32((uint16_t)((uint32_t)raw[i] >> 16));
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; i++) out[i] = ((const float *)w)[e + i];
  }
}

// e4m3 of a value: beyond the range the largest, but a NaN stays one
__device__ __forceinline__ float fp8_range(float v) { return v != v ? v : clamp_fp8(v); }
__device__ __forceinline__ v2i pack8_fp8(const float *v) {
  int lo = __builtin_amdgcn_cvt_pk_fp8_f32(fp8_range(v[0]), fp8_range(v[1]), 0, false);
  lo = __builtin_amdgcn_cvt_pk_fp8_f32(fp8_range(v[2]), fp8_range(v[3]), lo, true);
  int hi = __builtin_amdgcn_cvt_pk_fp8_f32(fp8_range(v[4]), fp8_range(v[5]), 0, false);
  hi = __builtin_amdgcn_cvt_pk_fp8_f32(fp8_range(v[6]), fp8_range(v[7]), hi, true);
  return (v2i){lo, hi};
}
__device__ __forceinline__ v2i scaled_fp8(const float *v, float scale) {
  float y[8];
#pragma unroll
  for (int i = 0; i < 8; i++) y[i] = v[i] / scale;
  return pack8_fp8(y);
}
__device__ __forceinline__ v4i pack8_bf16(const float *v) {
  return (v4i){(int)pack2_bf16(v[0], v[1]), (int)pack2_bf16(v[2], v[3]), (int)pack2_bf16(v[4], v[5]), (int)pack2_bf16(v[6], v[7])};
}

// 8 elements of a lane, 32 of four lanes side by side -> their codes and the byte of their power, 255 where one is no number.  In bits:
// a largest value of 2^k f with f up to 1.75 (4 f is at most 7) takes 2^(k - 2), above that 2^(k - 1); no more than 2^125, so that 6 of it is finite.
__device__ __forceinline__ uint32_t pack8_fp4(const float *v, uint32_t &power) {
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < 8; i++) top = max(top, __float_as_uint(v[i]) & 0x7fffffffu);       // (as whole numbers: NaN is above infinity)
  top = max(top, lane_xor<1>(top));
  top = max(top, lane_xor<2>(top));
  power = top >= 0x7f800000u ? 255u : (uint32_t)min(max((int)((top + 0x1fffffu) >> 23) - 2, 1), 252);
  const float p = __uint_as_float(min(power, 252u) << 23);
  uint32_t w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(0u, v[0], v[1], p, 0);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[2], v[3], p, 1);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[4], v[5], p, 2);
  return __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[6], v[7], p, 3);
}

template <int LPH, bool FOUR>                          // lanes of a head; a cache in 4 bits
__global__ __launch_bounds__(256) void qk_norm_rope_kernel(const RopeArgs a) {
  const int64_t group = (int64_t)blockIdx.x * (256 / LPH) + threadIdx.x / LPH;
  const int64_t t = group / a.groups_per_token;
  if (t >= a.T) return;                                // (whole groups of LPH lanes, which is what the shuffles reach)
  const int part = (int)(group % a.groups_per_token), L = threadIdx.x % LPH, e = 8 * L;
  const bool live = e < a.D;
  const int heads = a.Hq + 2 * a.Hkv;
  const int pos = a.positions[t];
  const bool placed = pos >= 0 && pos < a.P;
  const int64_t slot = a.slots ? a.slots[t] : -1;
  const bool stored = placed && slot >= 0 && slot < a.n_slots;
  const int half = a.R / 2, step = half / 8;           // lanes between the two of a pair
  const bool turned = live && e < a.R, second = e >= half;
  float c[8], s[8];
#pragma unroll
  for (int i = 0; i < 8; i++) c[i] = 1.f, s[i] = 0.f;
  if (turned && placed) {
    const float *row = a.cos_sin + (size_t)pos * a.R;
    if (a.interleaved) {
#pragma unroll
      for (int i = 0; i < 8; i++) c[i] = row[e / 2 + i / 2], s[i] = (i & 1) ? row[half + e / 2 + i / 2] : -row[half + e / 2 + i / 2];
    } else {
      const int f = second ? e - half : e;
#pragma unroll
      for (int i = 0; i < 8; i++) c[i] = row[f + i], s[i] = second ? row[half + f + i] : -row[half + f + i];
    }
  }
  const int lane = threadIdx.x & 63;
  const int other = turned && !a.interleaved ? (second ? lane - step : lane + step) : lane;
  const uint16_t *src = a.qkv + t * a.row_stride + e;
  const v4i none = (v4i){0, 0, 0, 0};

  // Of a query or key head: y = r (x w cos + x' w' sin), where x' and w' are the pair's other value and weight and r is 1 over the
  // root mean square.  w cos and w' sin are the same for all heads of a kind: formed once.
  float wc[8], ws[8];
  const auto factors = [&](const void *w) {
    float w1[8], w2[8];
#pragma unroll
    for (int i = 0; i < 8; i++) w1[i] = w2[i] = 1.f;
    if (w && live) {
      load_weight(w, a.weights_bf16, e, w1);
      load_weight(w, a.weights_bf16, e + 8 * (other - lane), w2);
    }
#pragma unroll
    for (int i = 0; i < 8; i++) wc[i] = w1[i] * c[i], ws[i] = (a.interleaved ? w1[i ^ 1] : w2[i]) * s[i];
  };
  const auto turn = [&](const v4i raw, bool normed, float (&y)[8]) {
    float x[8], z[8];
    float r = 1.f;
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const uint32_t o = a.interleaved ? (uint32_t)raw[i] : (uint32_t)__shfl(raw[i], other, 64);
      x[2 * i] = bf16_to_f32((uint16_t)((uint32_t)raw[i] & 0xffff));
      x[2 * i + 1] = bf16_to_f32((uint16_t)((uint32_t)raw[i] >> 16));
      const float lo = bf16_to_f32((uint16_t)(o & 0xffff)), hi = bf16_to_f32((uint16_t)(o >> 16));
      z[2 * i] = a.interleaved ? hi : lo;
      z[2 * i + 1] = a.interleaved ? lo : hi;
    }
    if (normed) {
      float sum = 0.f;
#pragma unroll
      for (int i = 0; i < 8; i++) sum = fmaf(x[i], x[i], sum);
      r = 1.0f / sqrtf(lane_sum<LPH>(sum) / (float)a.D + a.eps);
    }
#pragma unroll
    for (int i = 0; i < 8; i++) {
      const float o = x[i] * wc[i];
      y[i] = r * (turned ? fmaf(z[i], ws[i], o) : o);
    }
  };
  const auto place = [&](uint8_t *cache, int64_t block_bytes, int kh) {
    const int64_t within = ((slot & ((1 << a.page_log2) - 1)) * a.Hkv + kh) * (int64_t)a.D + e;
    return cache + (slot >> a.page_log2) * block_bytes + (FOUR ? within / 2 : within * (a.cache_fp8 ? 1 : 2));
  };
  const auto put4 = [&](uint8_t *cache, int64_t block_bytes, uint8_t *powers, int64_t powers_block, int kh, const float *v) {
    uint32_t power;
    const uint32_t w = pack8_fp4(v, power);
    *(uint32_t *)place(cache, block_bytes, kh) = w;
    if (L % 4 == 0) powers[(slot >> a.page_log2) * powers_block + ((slot & ((1 << a.page_log2) - 1)) * a.Hkv + kh) * (int64_t)(a.D / 32) + e / 32] = (uint8_t)power;
  };

  // Heads part, part + stride, ...: groups side by side read and write heads side by side.
  const int stride = a.groups_per_token;
  int h = part;
  float y[8];
  v4i raw = live && h < heads ? *(const v4i *)(src + (size_t)h * a.D) : none;
  const auto next = [&]() {                            // the next head is asked for before this one is worked on
    const v4i now = raw;
    h += stride;
    if (h < heads && live) raw = *(const v4i *)(src + (size_t)h * a.D);
    return now;
  };
  if (h < a.Hq) factors(a.q_weight);
  while (h < a.Hq) {
    uint16_t *at = a.q_out + (t * a.Hq + h) * a.D + e;
    turn(next(), a.q_weight != nullptr, y);
    if (live) *(v4i *)at = placed ? pack8_bf16(y) : none;
  }
  if (h < a.Hq + a.Hkv) factors(a.k_weight);
  while (h < a.Hq + a.Hkv) {
    const int kh = h - a.Hq;
    turn(next(), a.k_weight != nullptr, y);
    if (!live) continue;
    if (a.k_out) *(v4i *)(a.k_out + (t * a.Hkv + kh) * a.D + e) = placed ? pack8_bf16(y) : none;
    if (!a.k_cache || !stored) continue;
    if (FOUR) {
      put4(a.k_cache, a.k_block_bytes, a.k_powers, a.k_powers_block, kh, y);
      continue;
    }
    uint8_t *at = place(a.k_cache, a.k_block_bytes, kh);
    if (a.cache_fp8) *(v2i *)at = scaled_fp8(y, a.k_scale ? a.k_scale[kh] : 1.0f);
    else *(v4i *)at = pack8_bf16(y);
  }
  while (h < heads) {
    const int kh = h - a.Hq - a.Hkv;
    const v4i now = next();
    if (!live || !a.v_cache || !stored) continue;
    uint8_t *at = place(a.v_cache, a.v_block_bytes, kh);
    if (!FOUR && !a.cache_fp8) {
      *(v4i *)at = now;
      continue;
    }
#pragma unroll
    for (int i = 0; i < 4; i++) {
      y[2 * i] = bf16_to_f32((uint16_t)((uint32_t)now[i] & 0xffff));
      y[2 * i + 1] = bf16_to_f32((uint16_t)((uint32_t)now[i] >> 16));
    }
    if (FOUR) put4(a.v_cache, a.v_block_bytes, a.v_powers, a.v_powers_block, kh, y);
    else *(v2i *)at = scaled_fp8(y, a.v_scale ? a.v_scale[kh] : 1.0f);
  }
}

// Both entry points.  powers: of a cache in 4 bits (then cache_dtype is MOE_DTYPE_FP4).
static int norm_rope(void *stream, const void *qkv_bf16, int64_t row_stride, int T, int Hq, int Hkv, int D, const int32_t *positions,
                     const float *cos_sin, int P, int R, int interleaved, const void *q_weight, const void *k_weight, int weight_dtype, float eps,
                     void *q_out_bf16, void *k_out_bf16, void *k_cache, void *v_cache, int cache_dtype, int n_blocks, int64_t k_block_stride,
                     int64_t v_block_stride, int page_size, const int64_t *slots, const float *k_scale, const float *v_scale, uint8_t *k_powers,
                     uint8_t *v_powers, int64_t k_powers_block, int64_t v_powers_block) {
  const bool four = cache_dtype == MOE_DTYPE_FP4;
  if (T < 0 || Hq < 1 || Hkv < 1 || Hq > 4096 || Hkv > 4096 || D < 8 || D > 256 || P < 0 || R < 0 || R > D) return MOE_E_SHAPE;
  if (D % 8 || R % 16) return MOE_E_ALIGN;
  if (weight_dtype != MOE_DTYPE_F32 && weight_dtype != MOE_DTYPE_BF16) return MOE_E_MODE;
  const bool cached = k_cache || v_cache;
  if (cached) {
    if (cache_dtype != MOE_DTYPE_BF16 && cache_dtype != MOE_DTYPE_FP8 && !four) return MOE_E_MODE;
    const int64_t row = (int64_t)Hkv * D;
    if (n_blocks < 0 || page_size < 1 || page_size > MOE_MAX_PAGE || (page_size & (page_size - 1)) || k_block_stride < page_size * row ||
        v_block_stride < page_size * row)
      return MOE_E_SHAPE;
    if (four && (k_powers_block < page_size * row / 32 || v_powers_block < page_size * row / 32)) return MOE_E_SHAPE;
    if (k_block_stride % (four ? 32 : 8) || v_block_stride % (four ? 32 : 8)) return MOE_E_ALIGN;
  }
  const int64_t heads = (int64_t)Hq + 2 * Hkv;
  if (row_stride < heads * D) return MOE_E_SHAPE;
  if (row_stride % 8) return MOE_E_ALIGN;
  if (T == 0) return MOE_OK;
  if (!qkv_bf16 || !positions || (R && P && !cos_sin) || !q_out_bf16) return MOE_E_NULL;
  if (cached && (!k_cache || !v_cache || !slots || (four && (!k_powers || !v_powers)))) return MOE_E_NULL;
  for (const void *p : {qkv_bf16, q_weight, k_weight, (const void *)q_out_bf16, (const void *)k_out_bf16, (const void *)k_cache, (const void *)v_cache})
    if ((uintptr_t)p % 16) return MOE_E_ALIGN;
  const int wide = cached && cache_dtype == MOE_DTYPE_FP8 ? 1 : 2;
  RopeArgs a{(const uint16_t *)qkv_bf16, row_stride, positions, cos_sin, q_weight, k_weight, (uint16_t *)q_out_bf16, (uint16_t *)k_out_bf16,
             (uint8_t *)k_cache, (uint8_t *)v_cache, four ? k_block_stride / 2 : k_block_stride * wide, four ? v_block_stride / 2 : v_block_stride * wide,
             cached ? (int64_t)n_blocks * page_size : 0, cached ? slots : nullptr, k_scale, v_scale, k_powers, v_powers, k_powers_block, v_powers_block, eps, T, Hq, Hkv, D, R, P,
             cached ? __builtin_ctz(page_size) : 0, weight_dtype == MOE_DTYPE_BF16, interleaved ? 1 : 0, wide == 1, (int)heads};
  // A group's heads: one while the chip is not full of groups, then as many as leave 16384 of them (6000 tokens of 40 heads: 26 us, 31 with
  // 32768; 2500 into an e4m3 cache 16.6 and 18.1, 15.6 with 8192, which takes 613 tokens of 64-element heads from 4.8 to 6.1), at most 10 (16384
  // tokens: 5, 10, 20 heads take 80, 72, 75 to 81).
  const int64_t share = (int64_t)T * heads / 16384;
  const int64_t most = share < 1 ? 1 : share > 10 ? 10 : share;
  a.groups_per_token = (int)((heads + most - 1) / most);
  const int lph = D <= 32 ? 4 : D <= 64 ? 8 : D <= 128 ? 16 : 32;
  const int64_t groups = (int64_t)T * a.groups_per_token, blocks = (groups + 256 / lph - 1) / (256 / lph);
  if (blocks * 256 >> 32) return MOE_E_SHAPE;          // (a launch has fewer than 2^32 threads)
  hipStream_t st = (hipStream_t)stream;
  const auto run = [&](auto lanes) {
    constexpr int LPH = decltype(lanes)::value;
    if (four) qk_norm_rope_kernel<LPH, true><<<(unsigned)blocks, 256, 0, st>>>(a);
    else qk_norm_rope_kernel<LPH, false><<<(unsigned)blocks, 256, 0, st>>>(a);
  };
  if (lph == 4) run(std::integral_constant<int, 4>());
  else if (lph == 8) run(std::integral_constant<int, 8>());
  else if (lph == 16) run(std::integral_constant<int, 16>());
  else run(std::integral_constant<int, 32>());
  return (int)hipGetLastError();
}

}  // namespace moe

extern "C" int moe_qk_norm_rope(void *stream, const void *qkv_bf16, int64_t row_stride, int T, int Hq, int Hkv, int D,
                                const int32_t *positions, const float *cos_sin, int P, int R, int interleaved, const void *q_weight,
                                const void *k_weight, int weight_dtype, float eps, void *q_out_bf16, void *k_out_bf16, void *k_cache,
                                void *v_cache, int cache_dtype, int n_blocks, int64_t k_block_stride, int64_t v_block_stride,
                                int page_size, const int64_t *slots, const float *k_scale, const float *v_scale) {
  if ((k_cache || v_cache) && cache_dtype == MOE_DTYPE_FP4) cache_dtype = -1;             // (has no room for the powers: refused where modes are)
  return moe::norm_rope(stream, qkv_bf16, row_stride, T, Hq, Hkv, D, positions, cos_sin, P, R, interleaved, q_weight, k_weight, weight_dtype, eps,
                        q_out_bf16, k_out_bf16, k_cache, v_cache, cache_dtype, n_blocks, k_block_stride, v_block_stride, page_size, slots, k_scale,
                        v_scale, nullptr, nullptr, 0, 0);
}

extern "C" int moe_qk_norm_rope_fp4(void *stream, const void *qkv_bf16, int64_t row_stride, int T, int Hq, int Hkv, int D,
                                    const int32_t *positions, const float *cos_sin, int P, int R, int interleaved, const void *q_weight,
                                    const void *k_weight, int weight_dtype, float eps, void *q_out_bf16, void *k_cache, void *v_cache, int n_blocks,
                                    int64_t k_block_stride, int64_t v_block_stride, int page_size, const int64_t *slots, void *k_scale, void *v_scale,
                                    int64_t k_scale_block_stride, int64_t v_scale_block_stride) {
  if (D % 32) return MOE_E_ALIGN;
  if (T > 0 && (!k_cache || !v_cache)) return MOE_E_NULL;
  return moe::norm_rope(stream, qkv_bf16, row_stride, T, Hq, Hkv, D, positions, cos_sin, P, R, interleaved, q_weight, k_weight, weight_dtype, eps,
                        q_out_bf16, nullptr, k_cache, v_cache, MOE_DTYPE_FP4, n_blocks, k_block_stride, v_block_stride, page_size, slots, nullptr, nullptr,
                        (uint8_t *)k_scale, (uint8_t *)v_scale, k_scale_block_stride, v_scale_block_stride);
}
