// The products of MX4 matrices (moe_mx4_matmul_async, moe_mx4_linear_async).
#include "mx4.h"
#include "mx4_api.h"
#include "ops.h"

namespace c0ven {

// One wave a 16 x 16 tile of y: w's rows are the instruction's first operand, so that a lane holds four neighbours of a
// row of y.
template <uint32_t kType>
__global__ void __launch_bounds__(64) mx4_matmul(const uint8_t *xc, const uint8_t *xs, const uint8_t *wc,
                                                 const uint8_t *ws, uint32_t M, uint32_t N, uint32_t steps,
                                                 typename Elem<kType>::T *y, uint64_t stride) {
  const uint32_t lane = threadIdx.x, q = lane / 16, nt = (N + 15) / 16;
  const uint32_t n0 = blockIdx.x % nt * 16, m0 = blockIdx.x / nt * 16;
  const uint64_t wr = (uint64_t)min(n0 + lane % 16, N - 1) * steps, xr = (uint64_t)min(m0 + lane % 16, M - 1) * steps;
  mx_f4 c = {0, 0, 0, 0};
  for (uint32_t k = 0; k < steps; k++) {
    const mx_i4 a = *(const mx_i4 *)(wc + (wr + k) * 64 + q * 16), b = *(const mx_i4 *)(xc + (xr + k) * 64 + q * 16);
    c = mx_mfma16<0, 0>(a, b, c, ws[(wr + k) * 4 + q], xs[(xr + k) * 4 + q]);
  }
  const uint32_t m = m0 + lane % 16;
#pragma unroll
  for (uint32_t i = 0; i < 4; i++) {
    const uint32_t n = n0 + 4 * q + i;
    if (m < M && n < N) y[(uint64_t)m * stride + n] = (typename Elem<kType>::T)c[i];
  }
}

}  // namespace c0ven

using namespace c0ven;

namespace {

void launch_matmul(const uint8_t *xc, const uint8_t *xs, uint32_t M, const moe_mx4_matrix *w, uint32_t y_type, void *y,
                   uint64_t stride, void *stream) {
  const uint64_t n = (uint64_t)((M + 15) / 16) * ((w->rows + 15) / 16);
  const auto run = [&](auto kernel, auto *p) {
    op_launch(kernel, n, 64, stream, xc, xs, (const uint8_t *)w->codes, (const uint8_t *)w->scales, M, w->rows,
              mx_steps(w->cols), p, stride);
  };
  if (y_type == QT_F32) run(mx4_matmul<QT_F32>, (float *)y);
  if (y_type == QT_F16) run(mx4_matmul<QT_F16>, (_Float16 *)y);
  if (y_type == QT_BF16) run(mx4_matmul<QT_BF16>, (__bf16 *)y);
}

uint64_t quantised_bytes(uint32_t rows, uint32_t cols) { return moe_mx4_code_bytes(rows, cols) + (moe_mx4_scale_bytes(rows, cols) + 15) / 16 * 16; }

}  // namespace

extern "C" {

MOE_API uint64_t moe_mx4_matmul_work_bytes(const moe_mx4_matrix *, uint32_t) { return 0; }

MOE_API moe_status moe_mx4_matmul_async(int32_t device, const moe_mx4_matrix *x, const moe_mx4_matrix *w,
                                        uint32_t y_type, void *y, uint64_t y_stride, void *work, uint64_t work_bytes,
                                        void *stream) {
  return op_guarded([&] {
    op_mx4(x);
    op_mx4(w);
    op_require(x->cols == w->cols, "x and w must have the same cols");
    op_rows(y, y_stride, w->rows, y_type);
    op_work(work, work_bytes, moe_mx4_matmul_work_bytes(w, x->rows));
    OnDevice on(device);
    launch_matmul(x->codes, x->scales, x->rows, w, y_type, y, y_stride, stream);
  });
}

MOE_API uint64_t moe_mx4_linear_work_bytes(const moe_mx4_matrix *w, uint32_t ntok) {
  return w ? quantised_bytes(ntok, w->cols) : 0;
}

MOE_API moe_status moe_mx4_linear_async(int32_t device, uint32_t x_type, const void *x, uint64_t x_stride,
                                        uint32_t ntok, const moe_mx4_matrix *w, uint32_t y_type, void *y,
                                        uint64_t y_stride, void *work, uint64_t work_bytes, void *stream) {
  return op_guarded([&] {
    op_mx4(w);
    op_rows(x, x_stride, w->cols, x_type);
    op_rows(y, y_stride, w->rows, y_type);
    op_require(ntok <= 1u << 30, "too many tokens");
    op_work(work, work_bytes, moe_mx4_linear_work_bytes(w, ntok));
    if (!ntok) return;
    OnDevice on(device);
    uint8_t *xc = (uint8_t *)work, *xs = xc + moe_mx4_code_bytes(ntok, w->cols);
    const moe_mx4_matrix xm{xc, xs, ntok, w->cols};
    mx4_quantize_launch(x_type, x, x_stride, xm, stream);
    launch_matmul(xc, xs, ntok, w, y_type, y, y_stride, stream);
  });
}

}  // extern "C"
