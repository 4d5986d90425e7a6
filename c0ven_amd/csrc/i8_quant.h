// Rows of floats quantised to I8, from memory to memory.
#pragma once

#include "i8.h"

namespace c0ven {

// Rows of x to codes and scales, by work-group `block` of `blocks` of kBlock threads: kThreads threads a row (64, or all), kAhead
// groups of eight values a thread at a time. A row of that many is in registers, read once, so that the scale (the row's
// largest) is known before the codes are formed; kLong: longer rows, read again for their codes. Bound by memory: 4096 x 8192 of
// bf16 21.6 us, 4.7 TB/s, 16384 x 8192 71, 5.7; short rows, a wave each, by their number: 25915 x 100 9.1.
template <uint32_t kType, int kBlock, int kThreads, int kAhead, bool kLong>
__device__ __forceinline__ void quantize_block(uint32_t block, uint32_t blocks, const typename Elem<kType>::T *x, uint64_t stride,
                                               uint32_t rows, uint32_t cols, const uint32_t *n_rows, int8_t *codes, float *scales) {
  constexpr uint32_t kRows = kBlock / kThreads, kWaves = kThreads / 64, kSpan = kThreads * kAhead;
  __shared__ uint32_t most_of[2][kWaves];
  const uint32_t tid = threadIdx.x % kThreads, ng = i8_pitch(cols) / 8;
  if (n_rows) rows = min(rows, *n_rows);
  uint32_t turn = 0;
  for (uint32_t r0 = block * kRows; r0 < rows; r0 += blocks * kRows, turn ^= 1) {
    const uint32_t r = r0 + threadIdx.x / kThreads;
    if (kRows > 1 && r >= rows) break;  // (a wave's)
    const auto *row = x + r * stride;
    float v[kAhead][8];
    uint32_t most = 0;
    for (uint32_t g0 = tid; g0 < (kLong ? ng : tid + 1); g0 += kSpan) {
      load_eights<kType, kAhead>(cols, [&](int) { return row; }, [&](int i) { return (g0 + i * kThreads) * 8; }, v);
#pragma unroll
      for (int i = 0; i < kAhead; i++) most = max(most, most_of8(v[i]));
    }
#pragma unroll
    for (int m = 32; m >= 1; m /= 2) most = max(most, (uint32_t)__shfl_xor((int)most, m, 64));
    if (kWaves > 1) {
      if (threadIdx.x % 64 == 0) most_of[turn][threadIdx.x / 64] = most;
      __syncthreads();
#pragma unroll
      for (uint32_t w = 0; w < kWaves; w++) most = max(most, most_of[turn][w]);
    }
    const float s = i8_scale_of(most);
    for (uint32_t g0 = tid; g0 < (kLong ? ng : tid + 1); g0 += kSpan) {
      if (kLong) load_eights<kType, kAhead>(cols, [&](int) { return row; }, [&](int i) { return (g0 + i * kThreads) * 8; }, v);
#pragma unroll
      for (int i = 0; i < kAhead; i++) {
        const uint32_t g = g0 + i * kThreads;
        if (g < ng) *(uint2 *)(codes + (uint64_t)r * ng * 8 + g * 8) = i8_codes8(v[i], s);
      }
    }
    if (tid == 0) scales[r] = s;
  }
}

}  // namespace c0ven
