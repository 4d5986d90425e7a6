// Quantisation to 8-bit integers with a scale a row, and back (moe_i8_quantize_async, moe_i8_dequantize_async).
#include "i8_api.h"
#include "i8_quant.h"

#include <algorithm>

namespace c0ven {

template <uint32_t kType, int kThreads, int kAhead, bool kLong = false>
__global__ void __launch_bounds__(kThreads < 256 ? 256 : kThreads)
    i8_quantize(const typename Elem<kType>::T *x, uint64_t stride, uint32_t rows, uint32_t cols, const uint32_t *n_rows,
                int8_t *codes, float *scales) {
  quantize_block<kType, kThreads < 256 ? 256 : kThreads, kThreads, kAhead, kLong>(blockIdx.x, gridDim.x, x, stride, rows, cols, n_rows,
                                                                                 codes, scales);
}

// Eight values a thread: code * scale in fp32, then rounded to the type. Bound by memory: 4096 x 8192 to bf16 19.7 us, 5.1 TB/s, 16384 x
// 8192 70, 5.8; 25915 x 100 3.9.
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
