// Quantisation to microscaled 4-bit floats and back (moe_mx4_quantize_async, moe_mx4_dequantize_async).
#include "mx4.h"

#include "mx4_api.h"

#include <algorithm>

namespace c0ven {

// Both kernels take eight values a thread and kAhead such groups, all loaded before the first is used. A work-group has 256 /
// 2^shift rows of 2^shift threads (whole rows where they are short), each 2^shift kAhead groups wide. Bound by memory: 16384 x
// 8192 bf16 are quantised in 74 us (4.6 TB/s; with two groups a thread 77, four 83, eight 87), and back in 59 (5.8 TB/s) with
// four (two 69, eight 71).
struct MxRows {
  uint32_t rows, cols, shift, wide;  // wide: work-groups a row takes
};

template <uint32_t kType, int kAhead>
__global__ void __launch_bounds__(256) mx4_quantize(const typename Elem<kType>::T *x, uint64_t stride, MxRows a,
                                                    uint8_t *codes, uint8_t *scales) {
  const uint32_t ng = mx_steps(a.cols) * 16;
  const uint32_t r = (blockIdx.x / a.wide << (8 - a.shift)) + (threadIdx.x >> a.shift);
  const uint32_t g0 = (blockIdx.x % a.wide * kAhead << a.shift) + (threadIdx.x & ((1u << a.shift) - 1));
  if (r >= a.rows) return;  // (four neighbours of a block are in one row)
  const typename Elem<kType>::T *row = x + r * stride;
  float v[kAhead][8];
#pragma unroll
  for (int i = 0; i < kAhead; i++) load8<kType>(row, (g0 + (i << a.shift)) * 8, a.cols, v[i]);
#pragma unroll
  for (int i = 0; i < kAhead; i++) {
    const uint32_t g = g0 + (i << a.shift);
    uint32_t s;
    const uint32_t c = mx_quantize8(v[i], s);
    if (g >= ng) break;
    ((uint32_t *)codes)[(uint64_t)r * ng + g] = c;
    if (g % 4 == 0) scales[((uint64_t)r * ng + g) / 4] = (uint8_t)s;
  }
}

template <uint32_t kType, int kAhead>
__global__ void __launch_bounds__(256) mx4_dequantize(const uint8_t *codes, const uint8_t *scales, MxRows a,
                                                      typename Elem<kType>::T *out, uint64_t stride) {
  const uint32_t ng = mx_steps(a.cols) * 16;
  const uint32_t r = (blockIdx.x / a.wide << (8 - a.shift)) + (threadIdx.x >> a.shift);
  const uint32_t g0 = (blockIdx.x % a.wide * kAhead << a.shift) + (threadIdx.x & ((1u << a.shift) - 1));
  if (r >= a.rows) return;
  uint32_t c[kAhead], s[kAhead];
#pragma unroll
  for (int i = 0; i < kAhead; i++) {
    const uint64_t at = (uint64_t)r * ng + min(g0 + (i << a.shift), ng - 1);
    c[i] = ((const uint32_t *)codes)[at], s[i] = scales[at / 4];
  }
#pragma unroll
  for (int i = 0; i < kAhead; i++) {
    float v[8];
    mx_values8(c[i], mx_pow2(s[i]), v);
    store8<kType>(out + r * stride, (g0 + (i << a.shift)) * 8, a.cols, v);
  }
}

}  // namespace c0ven

using namespace c0ven;

namespace {

// launch(r0, rows' shape, work-groups) for the rows r0 and on, as many as a launch has threads for (less than 2^32; 2^27 rows of
// 129 values are two launches).
template <typename F>
void by_rows(uint32_t rows, uint32_t cols, uint32_t ahead, F launch) {
  const uint32_t ng = mx_steps(cols) * 16;
  uint32_t shift = 4;
  while (shift < 8 && ahead << shift < ng) shift++;
  const uint32_t wide = (ng + (ahead << shift) - 1) / (ahead << shift), per = 256 >> shift;
  const uint32_t most = ((1u << 24) - 1) / wide * per;
  for (uint32_t r0 = 0; r0 < rows; r0 += most) {
    const uint32_t n = std::min(rows - r0, most);
    launch(r0, MxRows{n, cols, shift, wide}, (uint64_t)(n + per - 1) / per * wide);
  }
}

}  // namespace

void c0ven::mx4_quantize_launch(uint32_t type, const void *x, uint64_t stride, const moe_mx4_matrix &m, void *stream) {
  by_rows(m.rows, m.cols, 1, [&](uint32_t r0, const MxRows &a, uint64_t n) {
    const auto run = [&](auto kernel, auto *p) {
      op_launch(kernel, n, 256, stream, p + r0 * stride, stride, a, m.codes + moe_mx4_code_bytes(r0, m.cols),
                m.scales + moe_mx4_scale_bytes(r0, m.cols));
    };
    if (type == QT_F32) run(mx4_quantize<QT_F32, 1>, (const float *)x);
    if (type == QT_F16) run(mx4_quantize<QT_F16, 1>, (const _Float16 *)x);
    if (type == QT_BF16) run(mx4_quantize<QT_BF16, 1>, (const __bf16 *)x);
  });
}

extern "C" {

MOE_API uint64_t moe_mx4_code_bytes(uint32_t rows, uint32_t cols) { return (uint64_t)rows * mx_steps(cols) * 64; }
MOE_API uint64_t moe_mx4_scale_bytes(uint32_t rows, uint32_t cols) { return (uint64_t)rows * mx_steps(cols) * 4; }

MOE_API moe_status moe_mx4_quantize_async(int32_t device, uint32_t type, const void *x, uint64_t stride,
                                          const moe_mx4_matrix *m, void *stream) {
  return op_guarded([&] {
    op_mx4(m);
    op_rows(x, stride, m->rows, m->cols, type);
    if (!m->rows) return;
    OnDevice on(device);
    mx4_quantize_launch(type, x, stride, *m, stream);
  });
}

MOE_API moe_status moe_mx4_dequantize_async(int32_t device, const moe_mx4_matrix *m, uint32_t type, void *out,
                                            uint64_t stride, void *stream) {
  return op_guarded([&] {
    op_mx4(m);
    op_rows(out, stride, m->rows, m->cols, type);
    if (!m->rows) return;
    OnDevice on(device);
    const auto go = [&](auto ahead) {
      constexpr int kAhead = decltype(ahead)::value;
      by_rows(m->rows, m->cols, kAhead, [&](uint32_t r0, const MxRows &a, uint64_t n) {
        const auto run = [&](auto kernel, auto *p) {
          op_launch(kernel, n, 256, stream, (const uint8_t *)m->codes + moe_mx4_code_bytes(r0, m->cols),
                    (const uint8_t *)m->scales + moe_mx4_scale_bytes(r0, m->cols), a, p + r0 * stride, stride);
        };
        if (type == QT_F32) run(mx4_dequantize<QT_F32, kAhead>, (float *)out);
        if (type == QT_F16) run(mx4_dequantize<QT_F16, kAhead>, (_Float16 *)out);
        if (type == QT_BF16) run(mx4_dequantize<QT_BF16, kAhead>, (__bf16 *)out);
      });
    };
    // (Rows too short for four groups a thread in sixteen threads leave threads without work: 25915 x 100 9.5 us, 4.7 with one.)
    if (mx_steps(m->cols) >= 4)
      go(std::integral_constant<int, 4>());
    else
      go(std::integral_constant<int, 1>());
  });
}

}  // extern "C"
