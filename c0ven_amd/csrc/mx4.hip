// Quantisation to microscaled 4-bit floats and back (moe_mx4_quantize_async, moe_mx4_dequantize_async).
#include "mx4.h"

#include "mx4_api.h"

namespace c0ven {

// One block of 32 values a thread.
template <uint32_t kType>
__global__ void mx4_quantize(const typename Elem<kType>::T *x, uint64_t stride, uint32_t rows, uint32_t cols,
                             uint8_t *codes, uint8_t *scales) {
  const uint32_t nb = mx_steps(cols) * 4;
  const uint64_t i = (uint64_t)blockIdx.x * blockDim.x + threadIdx.x;
  if (i >= (uint64_t)rows * nb) return;
  const uint64_t r = i / nb;
  const uint32_t b = (uint32_t)(i - r * nb);
  float v[32];
  uint32_t most = 0;
#pragma unroll
  for (uint32_t j = 0; j < 32; j++) {
    v[j] = b * 32 + j < cols ? (float)x[r * stride + b * 32 + j] : 0.0f;
    most = max(most, __float_as_uint(v[j]) & 0x7fffffffu);
  }
  const uint32_t s = mx_scale_of(most);
  uint32_t w[4];
#pragma unroll
  for (int j = 0; j < 4; j++) w[j] = s == 255 ? 0u : mx_codes8(v + 8 * j, s);
  *(uint4 *)(codes + i * 16) = make_uint4(w[0], w[1], w[2], w[3]);
  scales[i] = (uint8_t)s;
}

// Eight values a thread.
template <uint32_t kType>
__global__ void mx4_dequantize(const uint8_t *codes, const uint8_t *scales, uint32_t rows, uint32_t cols,
                               typename Elem<kType>::T *out, uint64_t stride) {
  const uint32_t nw = mx_steps(cols) * 16;
  const uint64_t i = (uint64_t)blockIdx.x * blockDim.x + threadIdx.x;
  if (i >= (uint64_t)rows * nw) return;
  const uint64_t r = i / nw;
  const uint32_t c = (uint32_t)(i - r * nw) * 8;
  const uint32_t w = ((const uint32_t *)codes)[i];
  const float s = mx_pow2(scales[i / 4]);
#pragma unroll
  for (uint32_t j = 0; j < 8; j++) {
    const uint32_t q = w >> (4 * j) & 15, m = q & 7;
    const float a = m < 2 ? 0.5f * (float)m : __uint_as_float(((m >> 1) + 126) << 23 | (m & 1) << 22);
    if (c + j < cols) out[r * stride + c + j] = (typename Elem<kType>::T)((q & 8 ? -a : a) * s);
  }
}

}  // namespace c0ven

using namespace c0ven;

void c0ven::mx4_quantize_launch(uint32_t type, const void *x, uint64_t stride, const moe_mx4_matrix &m, void *stream) {
  const uint64_t n = ((uint64_t)m.rows * mx_steps(m.cols) * 4 + 255) / 256;
  const auto run = [&](auto kernel, auto *p) { op_launch(kernel, n, 256, stream, p, stride, m.rows, m.cols, m.codes, m.scales); };
  if (type == QT_F32) run(mx4_quantize<QT_F32>, (const float *)x);
  if (type == QT_F16) run(mx4_quantize<QT_F16>, (const _Float16 *)x);
  if (type == QT_BF16) run(mx4_quantize<QT_BF16>, (const __bf16 *)x);
}

extern "C" {

MOE_API uint64_t moe_mx4_code_bytes(uint32_t rows, uint32_t cols) { return (uint64_t)rows * mx_steps(cols) * 64; }
MOE_API uint64_t moe_mx4_scale_bytes(uint32_t rows, uint32_t cols) { return (uint64_t)rows * mx_steps(cols) * 4; }

MOE_API moe_status moe_mx4_quantize_async(int32_t device, uint32_t type, const void *x, uint64_t stride,
                                          const moe_mx4_matrix *m, void *stream) {
  return op_guarded([&] {
    op_mx4(m);
    op_rows(x, stride, m->cols, type);
    OnDevice on(device);
    mx4_quantize_launch(type, x, stride, *m, stream);
  });
}

MOE_API moe_status moe_mx4_dequantize_async(int32_t device, const moe_mx4_matrix *m, uint32_t type, void *out,
                                            uint64_t stride, void *stream) {
  return op_guarded([&] {
    op_mx4(m);
    op_rows(out, stride, m->cols, type);
    OnDevice on(device);
    const uint64_t n = ((uint64_t)m->rows * mx_steps(m->cols) * 16 + 255) / 256;
    const auto run = [&](auto kernel, auto *p) {
      op_launch(kernel, n, 256, stream, (const uint8_t *)m->codes, (const uint8_t *)m->scales, m->rows, m->cols, p, stride);
    };
    if (type == QT_F32) run(mx4_dequantize<QT_F32>, (float *)out);
    if (type == QT_F16) run(mx4_dequantize<QT_F16>, (_Float16 *)out);
    if (type == QT_BF16) run(mx4_dequantize<QT_BF16>, (__bf16 *)out);
  });
}

}  // extern "C"
