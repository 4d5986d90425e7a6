// Rows of floats quantised to I8 into LDS by a work-group that uses them itself.
#pragma once

#include "i8.h"

namespace c0ven {

// Rows 0 .. n - 1 (row_of(i): a pointer to i's values; at most kGroups groups of eight of them a thread) to codes at lc, `lpitch`
// bytes apart, and the bits of their largest |x| at most_of: all threads, each group loaded once. A barrier before it if LDS was
// in use; it ends with one.
template <uint32_t kX, int kGroups, typename F>
__device__ __forceinline__ void quantize_rows(uint32_t n, uint32_t pitch, uint32_t cols, F row_of, uint8_t *lc, uint32_t lpitch,
                                              uint32_t *most_of) {
  const uint32_t per = pitch / 8, all = n * per;  // (16 neighbouring groups are of one row)
  float v[kGroups][8];
#pragma unroll
  for (int j = 0; j < kGroups; j++) {
    const uint32_t i = threadIdx.x + j * blockDim.x;
    if (j * blockDim.x >= all) break;
    if (i < all) load8<kX>(row_of(i / per), i % per * 8, cols, v[j]);
  }
  if (threadIdx.x < n) most_of[threadIdx.x] = 0;
  __syncthreads();
#pragma unroll
  for (int j = 0; j < kGroups; j++) {
    const uint32_t i = threadIdx.x + j * blockDim.x;
    if (j * blockDim.x >= all) break;
    if (i < all) {
      uint32_t m = most_of8(v[j]);
      m = max(m, dpp_u32<kDppXor1>(m));
      m = max(m, dpp_u32<kDppXor2>(m));
      m = max(m, dpp_u32<kDppHalfMirror>(m));
      m = max(m, dpp_u32<kDppMirror>(m));
      if (threadIdx.x % 16 == 0) atomicMax(most_of + i / per, m);
    }
  }
  __syncthreads();
#pragma unroll
  for (int j = 0; j < kGroups; j++) {
    const uint32_t i = threadIdx.x + j * blockDim.x;
    if (j * blockDim.x >= all) break;
    if (i < all) *(uint2 *)(lc + i / per * lpitch + i % per * 8) = i8_codes8(v[j], i8_scale_of(most_of[i / per]));
  }
  __syncthreads();
}

}  // namespace c0ven
