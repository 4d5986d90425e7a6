// The products of MX4 matrices (moe_mx4_matmul_async, moe_mx4_linear_async).
#include "mx4.h"
#include "mx4_api.h"
#include "mx4_gemm.h"
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

// A tile of y a work-group, k split into parts of `span` stages (256 each); part p's sums go to y + p * part.
template <uint32_t kType, int TM, int TN>
__global__ void __launch_bounds__(256, TM *TN > 8 ? 1 : 2)
    mx4_gemm(const uint8_t *xc, const uint8_t *xs, const uint8_t *wc, const uint8_t *ws, uint32_t M, uint32_t N,
             uint32_t steps, uint32_t span, typename Elem<kType>::T *y, uint64_t stride, uint64_t part) {
  typedef MxTile<TM, TN> Tile;
  constexpr int BM = Tile::BM, BN = Tile::BN;
  typedef typename Elem<kType>::T T;
  __shared__ typename Tile::Stage s0;
  __shared__ typename Tile::Stage s1;
  const uint32_t tm = (M + BM - 1) / BM, tn = (N + BN - 1) / BN, stages = (steps + 1) / 2;
  const uint32_t parts = (stages + span - 1) / span, all = tm * tn * parts;
  const uint32_t per = (all + 7) / 8, id = blockIdx.x % 8 * per + blockIdx.x / 8;
  if (blockIdx.x / 8 >= per || id >= all) return;
  const uint32_t p = id / (tm * tn), t = id % (tm * tn), group = t / (8 * tn), rows = min(tm - group * 8, 8u);
  const uint32_t m0 = (group * 8 + t % (8 * tn) % rows) * BM, n0 = t % (8 * tn) / rows * BN;
  const uint32_t k0 = p * span, k1 = min(k0 + span, stages);
  const MxSource<BM> sx(xc, xs, m0, M, steps);
  const MxSource<BN> sw(wc, ws, n0, N, steps);
  const auto load = [&](typename Tile::Stage &s, uint32_t k) {
    sx.load(k, s.x, s.sx);
    sw.load(k, s.w, s.sw);
  };
  Tile c;
  c.clear();
  load(s0, k0);
  if (k0 + 1 < k1) load(s1, k0 + 1);
  dma_barrier();
  c.template read<0>(s0);
  c.template read_scales<0>(s0);
  for (uint32_t k = k0;; k += 2) {
    c.template stage<0>(s0, s1, 2 * k + 1 >= steps, [&] {
      if (k + 2 < k1) load(s0, k + 2);
    });
    if (k + 1 >= k1) break;
    c.template stage<1>(s1, s0, 2 * k + 3 >= steps, [&] {
      if (k + 3 < k1) load(s1, k + 3);
    });
    if (k + 2 >= k1) break;
  }
  __builtin_amdgcn_s_barrier();  // (the stages' LDS is used again)
  // Each wave's 32 rows at a time through its part of LDS, so that a row's neighbours are stored together.
  const uint32_t lane = threadIdx.x & 63, wave = mx_wave(), q = lane / 32, r = lane % 32;
  constexpr uint32_t kWide = 32 * TN, kPitch = kWide + 4;
  float *mine = (float *)(wave < 2 ? (uint8_t *)&s0 : (uint8_t *)&s1) + (wave & 1) * 32 * kPitch;
  static_assert(2 * 32 * kPitch * 4 <= sizeof(s0), "two waves' rows in a stage");
  const uint32_t wm = m0 + (wave & 1) * 32 * TM, wn = n0 + (wave >> 1) * kWide;
  y += p * part;
  const bool whole = wn + kWide <= N && stride % 4 == 0 && ((uintptr_t)y & (4 * sizeof(T) - 1)) == 0;
#pragma unroll
  for (int m = 0; m < TM; m++) {
#pragma unroll
    for (int n = 0; n < TN; n++)
#pragma unroll
      for (int j = 0; j < 4; j++)
        *(float4 *)(mine + r * kPitch + 32 * n + 8 * j + 4 * q) =
            make_float4(c.acc[n][m][4 * j], c.acc[n][m][4 * j + 1], c.acc[n][m][4 * j + 2], c.acc[n][m][4 * j + 3]);
    __builtin_amdgcn_s_waitcnt(0xc07f);
    __builtin_amdgcn_wave_barrier();
#pragma unroll 4
    for (uint32_t i = lane; i < 32 * kWide / 4; i += 64) {
      const uint32_t row = i / (kWide / 4), col = i % (kWide / 4) * 4;
      const float4 v = *(const float4 *)(mine + row * kPitch + col);
      const uint32_t gm = wm + 32 * m + row, gn = wn + col;
      T *to = y + (uint64_t)gm * stride + gn;
      const float e[4] = {v.x, v.y, v.z, v.w};
      if (gm >= M) continue;
      if (whole) {
        struct alignas(4 * sizeof(T)) Four {
          T e[4];
        };
        *(Four *)to = Four{{(T)v.x, (T)v.y, (T)v.z, (T)v.w}};
      } else {
        for (uint32_t j = 0; j < 4; j++)
          if (gn + j < N) to[j] = (T)e[j];
      }
    }
    __builtin_amdgcn_s_waitcnt(0xc07f);
    __builtin_amdgcn_wave_barrier();
  }
}

}  // namespace c0ven

using namespace c0ven;

namespace {

void launch_matmul(const uint8_t *xc, const uint8_t *xs, uint32_t M, const moe_mx4_matrix *w, uint32_t y_type, void *y,
                   uint64_t stride, void *stream) {
  const uint32_t N = w->rows, steps = mx_steps(w->cols);
  if (M >= 256 && N >= 256) {
    const uint64_t blocks = ((uint64_t)((M + 255) / 256) * ((N + 255) / 256) + 7) / 8 * 8;
    const auto gemm = [&](auto kernel, auto *p) {
      op_launch(kernel, blocks, 256, stream, xc, xs, (const uint8_t *)w->codes, (const uint8_t *)w->scales, M, N, steps,
                (steps + 1) / 2, p, stride, (uint64_t)0);
    };
    if (y_type == QT_F32) gemm(mx4_gemm<QT_F32, 4, 4>, (float *)y);
    if (y_type == QT_F16) gemm(mx4_gemm<QT_F16, 4, 4>, (_Float16 *)y);
    if (y_type == QT_BF16) gemm(mx4_gemm<QT_BF16, 4, 4>, (__bf16 *)y);
    return;
  }
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
