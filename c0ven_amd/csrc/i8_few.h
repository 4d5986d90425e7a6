// Rows of floats quantised to I8 into LDS by a work-group that uses them itself.
#pragma once

#include "i8.h"

namespace c0ven {

// Every wave is here, and what they wrote to and read from LDS is done; loads into LDS may be on their way (a fence would wait).
__device__ __forceinline__ void all_waves() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt(0xc07f);  // lgkmcnt(0)
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

// Rows 0 .. n - 1 of at least eight values (row_of(i): a pointer to i's) to codes, eight at a time to to(i, column), and the bits of
// their largest |x| to most_of; all threads. kAhead groups of eight values a thread at a time; more than that are read twice, the second
// time from the cache. It ends with a barrier. Little code: a work-group that comes this way once waits for its code as long as for
// its data (unrolled over twelve groups, 35 KB in all, one token's experts took 26 us).
template <uint32_t kX, int kAhead, typename Row, typename To>
__device__ __forceinline__ void quantize_rows(uint32_t n, uint32_t pitch, uint32_t cols, Row row_of, To to, uint32_t *most_of) {
  const uint32_t per = pitch / 8, all = n * per, round = kAhead * blockDim.x;  // (16 neighbouring groups are of one row)
  float v[kAhead][8];
  if (threadIdx.x < n) most_of[threadIdx.x] = 0;
  all_waves();
#pragma unroll 1
  for (uint32_t pass = 0; pass < 2; pass++) {
#pragma unroll 1
    for (uint32_t i0 = threadIdx.x; i0 < all; i0 += round) {
      uint32_t r[kAhead], c[kAhead];
#pragma unroll
      for (int j = 0; j < kAhead; j++) {
        const uint32_t i = min(i0 + j * blockDim.x, all - 1);
        r[j] = i / per, c[j] = (i - r[j] * per) * 8;
      }
      if (pass == 0 || all > round) {
        Eight<kX> e[kAhead];
#pragma unroll
        for (int j = 0; j < kAhead; j++) e[j].load(row_of(r[j]), c[j], cols);
#pragma unroll
        for (int j = 0; j < kAhead; j++) e[j].values(c[j], cols, v[j]);
      }
#pragma unroll
      for (int j = 0; j < kAhead; j++) {
        if (i0 + j * blockDim.x >= all) break;
        if (pass == 0) {
          uint32_t m = most_of8(v[j]);
          m = max(m, dpp_u32<kDppXor1>(m));
          m = max(m, dpp_u32<kDppXor2>(m));
          m = max(m, dpp_u32<kDppHalfMirror>(m));
          m = max(m, dpp_u32<kDppMirror>(m));
          if (threadIdx.x % 16 == 0) atomicMax(most_of + r[j], m);
        } else {
          *(uint2 *)to(r[j], c[j]) = i8_codes8(v[j], i8_scale_of(most_of[r[j]]));
        }
      }
    }
    all_waves();
  }
}

}  // namespace c0ven
