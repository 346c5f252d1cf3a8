// Moves between the lanes of a wave.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

// Value of v held by lane (lane ^ s) of the wave, s in {1, 2, 4, 8, 16, 32}
// (a compile-time constant after unrolling).  Cross-lane moves on the VALU:
// DPP quad permutes (1, 2), row shifts under bank masks (4), a row rotate
// (8), and gfx950's permlane16/permlane32 swaps (16, 32) -- no LDS round
// trip, unlike ds_bpermute.  Every lane of the wave must be active.
__device__ __forceinline__ uint32_t mxm_xor_lane(uint32_t v, int s) {
  const int lane = threadIdx.x & 63;
  switch (s) {
    case 1:
      return __builtin_amdgcn_update_dpp(0u, v, 0xB1, 0xf, 0xf, false);  // quad_perm [1,0,3,2]
    case 2:
      return __builtin_amdgcn_update_dpp(0u, v, 0x4E, 0xf, 0xf, false);  // quad_perm [2,3,0,1]
    case 4: {
      const uint32_t r = __builtin_amdgcn_update_dpp(0u, v, 0x104, 0xf, 0x5, false);  // row_shl:4
      return __builtin_amdgcn_update_dpp(r, v, 0x114, 0xf, 0xa, false);              // row_shr:4
    }
    case 8:
      return __builtin_amdgcn_update_dpp(0u, v, 0x128, 0xf, 0xf, false);  // row_ror:8
    case 16: {
      const auto r = __builtin_amdgcn_permlane16_swap(v, v, false, false);
      return (lane & 16) ? r[0] : r[1];
    }
    default: {
      const auto r = __builtin_amdgcn_permlane32_swap(v, v, false, false);
      return (lane & 32) ? r[0] : r[1];
    }
  }
}
__device__ __forceinline__ float mxm_xor_lane_f(float v, int s) {
  return __builtin_bit_cast(float, mxm_xor_lane(__builtin_bit_cast(uint32_t, v), s));
}
__device__ __forceinline__ int mxm_xor_lane_i(int v, int s) {
  return (int)mxm_xor_lane((uint32_t)v, s);
}
