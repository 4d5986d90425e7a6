// What the experts' kernels share whatever their weights' format.
#pragma once

#include "mx4.h"

namespace c0ven {

// silu(g) u with the limit of moe_config.swiglu_limit; NaNs stay.
__device__ __forceinline__ float expert_swiglu(float g, float u, float limit) {
  if (limit > 0.0f) {
    g = g > limit ? limit : g;
    u = u > limit ? limit : u < -limit ? -limit : u;
  }
  return g / (1.0f + exp_f32(-g)) * u;
}

// What lane l of 64 holds (flag) as the number of lanes below it that do.
__device__ __forceinline__ uint32_t lanes_below(uint64_t ballot) {
  return __builtin_amdgcn_mbcnt_hi((uint32_t)(ballot >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)ballot, 0u));
}

// A launch's work-groups to its items (parts a tile) so that an XCD (work-groups go to the eight in turn) has runs of four
// tiles: an expert's tiles share its weights in that L2, while the experts with one tile are dealt over all of them (MX4, 4096
// tokens of 10 of 512 experts 392 us, with the items in order 430; of 4 of 16 experts 114 and 119). ~0: none.
constexpr uint32_t kTileRun = 4;
__device__ __forceinline__ uint32_t item_of(uint32_t all, uint32_t parts, uint32_t j = blockIdx.x / 8) {
  const uint32_t run = kTileRun * parts, id = (j / run * 8 + blockIdx.x % 8) * run + j % run;
  return id < all ? id : ~0u;
}
// The work-groups that cover `all` items.
inline uint64_t item_blocks(uint64_t all, uint64_t parts) {
  const uint64_t run = kTileRun * parts;
  return (all + 8 * run - 1) / (8 * run) * (8 * run);
}

}  // namespace c0ven
