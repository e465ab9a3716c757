// Exchanges between the 16-lane groups of a wavefront, shared by the attention kernels.
#pragma once

#include "common.h"

namespace vdnh3 {

// Reductions over the four 16-lane groups of a wavefront through v_permlane32_swap / v_permlane16_swap (gfx950).
// lanes < 32: max of a over lane groups (g, g + 2); lanes >= 32: the same of b
__device__ __forceinline__ float max_pair32(float a, float b) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(a), __float_as_uint(b), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
// a over the four lane groups, b over the four lane groups, each in every lane
__device__ __forceinline__ void group_max(float &a, float &b) {
  const uint32_t x = __float_as_uint(max_pair32(a, b));
  const auto r = __builtin_amdgcn_permlane16_swap(x, x, false, false);
  const uint32_t y = __float_as_uint(fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1])));
  const auto q = __builtin_amdgcn_permlane32_swap(y, y, false, false);
  a = __uint_as_float(q[0]);
  b = __uint_as_float(q[1]);
}

}  // namespace vdnh3
