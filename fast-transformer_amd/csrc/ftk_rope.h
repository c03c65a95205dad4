// Lane exchanges of a head held by D / 8 neighbouring lanes, 8 elements each (the RoPE kernels).
#pragma once

#include "ftk_device.h"

namespace ftk {

// The pair of lane l ^ (LANES / 2) of each group of LANES lanes (16 or 8). row_ror:8 is l ^ 8 within 16
// lanes; row_half_mirror (7 - l) and then quad_perm [3,2,1,0] (l ^ 3) together are l ^ 4 within 8.
template <int LANES>
__device__ __forceinline__ uint32_t half_partner(uint32_t v) {
  if constexpr (LANES == 16) return dpp_u32<0x128, 0xF>(v);
  return dpp_u32<0x1B, 0xF>(dpp_u32<0x141, 0xF>(v));
}

// Sum over each group of LANES lanes, the same bits in all of them. For 16 lanes the order of the chunks
// is quad_group_sum's (^ 2, ^ 1, ^ 4, ^ 8), so a head is scaled as the fused attention prologue scales it.
template <int LANES>
__device__ __forceinline__ float head_sum(float v) {
  v += dpp<0x4E, 0xF>(v);   // quad_perm [2,3,0,1]: ^ 2
  v += dpp<0xB1, 0xF>(v);   // quad_perm [1,0,3,2]: ^ 1
  v += dpp<0x141, 0xF>(v);  // row_half_mirror: the other four of the eight
  if constexpr (LANES == 16) v += dpp<0x128, 0xF>(v);
  return v;
}

}  // namespace ftk
