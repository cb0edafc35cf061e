// Values of other lanes of a wavefront without a trip through LDS: data-parallel moves within rows of 16, row swaps across them.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace moe {

// the value of lane ^ D
template <int D>
__device__ __forceinline__ uint32_t lane_xor(uint32_t v) {
  static_assert(D == 1 || D == 2 || D == 4 || D == 8 || D == 16 || D == 32, "a power of two");
  typedef uint32_t v2u __attribute__((ext_vector_type(2)));
  if (D == 1) return __builtin_amdgcn_update_dpp(v, v, 0xb1, 0xf, 0xf, false);         // quad_perm 1 0 3 2
  if (D == 2) return __builtin_amdgcn_update_dpp(v, v, 0x4e, 0xf, 0xf, false);         // quad_perm 2 3 0 1
  if (D == 4) {                                                                        // from 4 lanes up and down in a row
    const uint32_t up = __builtin_amdgcn_update_dpp(v, v, 0x104, 0xf, 0x5, false);
    return __builtin_amdgcn_update_dpp(up, v, 0x114, 0xf, 0xa, false);
  }
  if (D == 8) return __builtin_amdgcn_update_dpp(v, v, 0x128, 0xf, 0xf, false);        // row rotated by 8
  const v2u r = D == 16 ? __builtin_amdgcn_permlane16_swap(v, v, false, false) : __builtin_amdgcn_permlane32_swap(v, v, false, false);
  return (threadIdx.x & D) ? r[0] : r[1];
}
template <int D>
__device__ __forceinline__ uint64_t lane_xor(uint64_t v) {
  return (uint64_t)lane_xor<D>((uint32_t)(v >> 32)) << 32 | lane_xor<D>((uint32_t)v);
}
template <int D>
__device__ __forceinline__ float lane_xor(float v) { return __uint_as_float(lane_xor<D>(__float_as_uint(v))); }

// the sum over LANES neighbouring lanes, a power of two
template <int LANES>
__device__ __forceinline__ float lane_sum(float v) {
  if constexpr (LANES > 1) {
    v = lane_sum<LANES / 2>(v);
    v += lane_xor<LANES / 2>(v);
  }
  return v;
}

// the sum of a wavefront's lanes 0 .. this one, 2^32 - 1 where it is more
__device__ __forceinline__ uint32_t lane_sum_upto(uint32_t v) {
  const auto add = [](uint32_t a, int b) { return __builtin_elementwise_add_sat(a, (uint32_t)b); };
  v = add(v, __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, false));               // from 1, 2, 4, 8 lanes down in a row of 16
  v = add(v, __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, false));
  v = add(v, __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, false));
  v = add(v, __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, false));
  v = add(v, __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false));               // a row's last lane to the next row
  return add(v, __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false));            // lane 31 to the upper half
}
// the largest over a wavefront
__device__ __forceinline__ int lane_max(int v) {
  v = max(v, (int)lane_xor<1>((uint32_t)v));
  v = max(v, (int)lane_xor<2>((uint32_t)v));
  v = max(v, (int)lane_xor<4>((uint32_t)v));
  v = max(v, (int)lane_xor<8>((uint32_t)v));
  v = max(v, (int)lane_xor<16>((uint32_t)v));
  return max(v, (int)lane_xor<32>((uint32_t)v));
}

}  // namespace moe
