// Sums and maxima over the lanes of a wavefront by moves between lanes: no trip to LDS.
#pragma once
#include <hip/hip_runtime.h>

namespace shainet {

// Over the lanes up to and with this one, of integers that are not negative (lanes without a source count as 0).
template <typename F>
__device__ __forceinline__ int scan_lanes(int x, F two) {
  x = two(x, __builtin_amdgcn_update_dpp(0, x, 0x111, 0xf, 0xf, false));  // row_shr 1, 2, 4, 8
  x = two(x, __builtin_amdgcn_update_dpp(0, x, 0x112, 0xf, 0xf, false));
  x = two(x, __builtin_amdgcn_update_dpp(0, x, 0x114, 0xf, 0xf, false));
  x = two(x, __builtin_amdgcn_update_dpp(0, x, 0x118, 0xf, 0xf, false));
  x = two(x, __builtin_amdgcn_update_dpp(0, x, 0x142, 0xa, 0xf, false));  // row_bcast 15, 31
  return two(x, __builtin_amdgcn_update_dpp(0, x, 0x143, 0xc, 0xf, false));
}
__device__ __forceinline__ int sum_lanes(int x) {
  return scan_lanes(x, [](int a, int b) { return a + b; });
}
__device__ __forceinline__ int max_lanes(int x) {
  return scan_lanes(x, [](int a, int b) { return max(a, b); });
}

}  // namespace shainet
