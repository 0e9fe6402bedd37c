// Sums over aligned groups of 2 to 64 lanes of a wavefront, in all lanes of the group: moves inside rows of 16 lanes, then
// exchanges of rows and of halves, and no LDS.  All 64 lanes must be active.
#ifndef MLUOP_AMD_CORE_LANE_SUM_H_
#define MLUOP_AMD_CORE_LANE_SUM_H_

#include <hip/hip_runtime.h>

#include <cstdint>

namespace mluop {

template <int CTRL>
__device__ __forceinline__ float lanesMoved(float v) {
  return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, 0xf, 0xf, true));
}

template <int LANES>
__device__ __forceinline__ float sumOverLanes(float v) {
  static_assert(LANES >= 1 && LANES <= 64 && (LANES & (LANES - 1)) == 0, "a power of two");
  if constexpr (LANES >= 2) v += lanesMoved<0xB1>(v);   // lanes 1 0 3 2 of every four
  if constexpr (LANES >= 4) v += lanesMoved<0x4E>(v);   // lanes 2 3 0 1
  if constexpr (LANES >= 8) v += lanesMoved<0x141>(v);  // the other four of eight, in mirrored order
  if constexpr (LANES >= 16) v += lanesMoved<0x140>(v); // the other eight of sixteen
  if constexpr (LANES >= 32) {
    // (rows 1 and 3 of the first word change places with rows 0 and 2 of the second)
    const auto rows = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = __uint_as_float(rows[0]) + __uint_as_float(rows[1]);
  }
  if constexpr (LANES >= 64) {
    const auto halves = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = __uint_as_float(halves[0]) + __uint_as_float(halves[1]);
  }
  return v;
}

}  // namespace mluop

#endif  // MLUOP_AMD_CORE_LANE_SUM_H_
