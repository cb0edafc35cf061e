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

}  // namespace moe
