// Quantisation to 8-bit integers with a scale a row, and back (moe_i8_quantize_async, moe_i8_dequantize_async).
#include "i8_api.h"

#include <algorithm>

namespace c0ven {

// kThreads threads a row (64: four rows a work-group), kAhead groups of eight values a thread at a time. A row of that many is in
// registers, read once, so that the scale (the row's largest) is known before the codes are formed; kLong: longer rows, read
// again for their codes. Bound by memory.
template <uint32_t kType, int kThreads, int kAhead, bool kLong = false>
__global__ void __launch_bounds__(kThreads < 256 ? 256 : kThreads)
    i8_quantize(const typename Elem<kType>::T *x, uint64_t stride, uint32_t rows, uint32_t cols, const uint32_t *n_rows,
                int8_t *codes, float *scales) {
  constexpr uint32_t kRows = kThreads < 256 ? 256 / kThreads : 1, kWaves = kThreads / 64, kSpan = kThreads * kAhead;
  __shared__ uint32_t most_of[2][kWaves];
  const uint32_t tid = threadIdx.x % kThreads, ng = i8_pitch(cols) / 8;
  if (n_rows) rows = min(rows, *n_rows);
  uint32_t turn = 0;
  for (uint32_t r0 = blockIdx.x * kRows; r0 < rows; r0 += gridDim.x * kRows, turn ^= 1) {
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

// Eight values a thread.
template <uint32_t kType>
__global__ void __launch_bounds__(256) i8_dequantize(const int8_t *codes, const float *scales, uint32_t rows, uint32_t cols,
                                                     typename Elem<kType>::T *out, uint64_t stride) {
  const uint32_t per = (cols + 7) / 8;
  const uint64_t n = (uint64_t)rows * per;
  for (uint64_t i = (uint64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (uint64_t)gridDim.x * 256) {
    const uint32_t r = (uint32_t)(i / per), g = (uint32_t)(i - (uint64_t)r * per);
    const uint2 c = *(const uint2 *)(codes + (uint64_t)r * i8_pitch(cols) + g * 8);
    const float s = scales[r];
    float v[8];
#pragma unroll
    for (int j = 0; j < 8; j++) v[j] = (float)(int8_t)((j < 4 ? c.x : c.y) >> (8 * (j % 4))) * s;
    store8<kType>(out + r * stride, g * 8, cols, v);
  }
}

constexpr uint64_t kMostBlocks = 1 << 16;  // (more rows go through them in turn)

void i8_quantize_launch(uint32_t type, const void *x, uint64_t stride, const moe_i8_matrix &m, const uint32_t *n_rows,
                        void *stream) {
  op_by_type(type, [&](auto t) {
    constexpr uint32_t kType = decltype(t)::value;
    const auto run = [&](auto kernel, uint32_t threads) {
      const uint32_t per = threads < 256 ? 256 / threads : 1;
      op_launch(kernel, std::min(((uint64_t)m.rows + per - 1) / per, kMostBlocks), std::max(threads, 256u), stream,
                (const typename Elem<kType>::T *)x, stride, m.rows, m.cols, n_rows, m.codes, m.scales);
    };
    const uint32_t groups = i8_pitch(m.cols) / 8;
    if (groups <= 64) run(i8_quantize<kType, 64, 1>, 64);
    else if (groups <= 256) run(i8_quantize<kType, 64, 4>, 64);
    else if (groups <= 1024) run(i8_quantize<kType, 256, 4>, 256);
    else if (groups <= 2048) run(i8_quantize<kType, 256, 8>, 256);
    else run(i8_quantize<kType, 1024, 4, true>, 1024);
  });
}

}  // namespace c0ven

using namespace c0ven;

extern "C" {

MOE_API uint64_t moe_i8_code_bytes(uint32_t rows, uint32_t cols) { return i8_bytes(rows, cols); }

MOE_API moe_status moe_i8_quantize_async(int32_t device, uint32_t type, const void *x, uint64_t stride, const moe_i8_matrix *m,
                                         void *stream) {
  return op_guarded([&] {
    op_i8(m);
    op_rows(x, stride, m->rows, m->cols, type);
    if (!m->rows) return;
    OnDevice on(device);
    i8_quantize_launch(type, x, stride, *m, nullptr, stream);
  });
}

MOE_API moe_status moe_i8_dequantize_async(int32_t device, const moe_i8_matrix *m, uint32_t type, void *out, uint64_t stride,
                                           void *stream) {
  return op_guarded([&] {
    op_i8(m);
    op_rows(out, stride, m->rows, m->cols, type);
    if (!m->rows) return;
    OnDevice on(device);
    const uint64_t n = (uint64_t)m->rows * ((m->cols + 7) / 8);
    op_by_type(type, [&](auto t) {
      constexpr uint32_t kType = decltype(t)::value;
      op_launch(i8_dequantize<kType>, std::min((n + 255) / 256, kMostBlocks), 256, stream, (const int8_t *)m->codes,
                (const float *)m->scales, m->rows, m->cols, (typename Elem<kType>::T *)out, stride);
    });
  });
}

}  // extern "C"
