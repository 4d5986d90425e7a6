// The experts of routed tokens in MX4 (moe_mx4_experts_async).
#include "mx4.h"
#include "mx4_api.h"
#include "ops.h"

namespace c0ven {

// silu(g) u with the limit of moe_config.swiglu_limit; NaNs stay.
__device__ __forceinline__ float mx_swiglu(float g, float u, float limit) {
  if (limit > 0.0f) {
    g = g > limit ? limit : g;
    u = u > limit ? limit : u < -limit ? -limit : u;
  }
  return g / (1.0f + expf(-g)) * u;
}

// One wave 16 rows of an assignment's expert.
__global__ void __launch_bounds__(64) mx4_gate_up(const uint8_t *xc, const uint8_t *xs, const uint8_t *gc,
                                                  const uint8_t *gs, const uint8_t *uc, const uint8_t *us,
                                                  const int32_t *ids, uint32_t E, uint32_t K, uint32_t H, uint32_t F,
                                                  float limit, float *h) {
  const uint32_t lane = threadIdx.x, q = lane / 16, nt = (F + 15) / 16, steps = mx_steps(H);
  const uint32_t a = blockIdx.x / nt, f0 = blockIdx.x % nt * 16;
  const uint32_t e = (uint32_t)ids[a];
  if (e >= E) return;
  const uint64_t wr = ((uint64_t)e * F + min(f0 + lane % 16, F - 1)) * steps, xr = (uint64_t)(a / K) * steps;
  mx_f4 g = {0, 0, 0, 0}, u = g;
  for (uint32_t k = 0; k < steps; k++) {
    const mx_i4 x = *(const mx_i4 *)(xc + (xr + k) * 64 + q * 16);
    const uint32_t sx = xs[(xr + k) * 4 + q];
    g = mx_mfma16<0, 0>(*(const mx_i4 *)(gc + (wr + k) * 64 + q * 16), x, g, gs[(wr + k) * 4 + q], sx);
    u = mx_mfma16<0, 0>(*(const mx_i4 *)(uc + (wr + k) * 64 + q * 16), x, u, us[(wr + k) * 4 + q], sx);
  }
  if (lane % 16 == 0)
#pragma unroll
    for (uint32_t i = 0; i < 4; i++)
      if (f0 + 4 * q + i < F) h[(uint64_t)a * F + f0 + 4 * q + i] = mx_swiglu(g[i], u[i], limit);
}

__global__ void __launch_bounds__(64) mx4_down(const uint8_t *hc, const uint8_t *hs, const uint8_t *dc,
                                               const uint8_t *ds, const int32_t *ids, uint32_t E, uint32_t H, uint32_t F,
                                               float *o) {
  const uint32_t lane = threadIdx.x, q = lane / 16, nt = (H + 15) / 16, steps = mx_steps(F);
  const uint32_t a = blockIdx.x / nt, r0 = blockIdx.x % nt * 16;
  const uint32_t e = (uint32_t)ids[a];
  if (e >= E) return;
  const uint64_t wr = ((uint64_t)e * H + min(r0 + lane % 16, H - 1)) * steps, xr = (uint64_t)a * steps;
  mx_f4 c = {0, 0, 0, 0};
  for (uint32_t k = 0; k < steps; k++)
    c = mx_mfma16<0, 0>(*(const mx_i4 *)(dc + (wr + k) * 64 + q * 16), *(const mx_i4 *)(hc + (xr + k) * 64 + q * 16), c,
                        ds[(wr + k) * 4 + q], hs[(xr + k) * 4 + q]);
  if (lane % 16 == 0)
#pragma unroll
    for (uint32_t i = 0; i < 4; i++)
      if (r0 + 4 * q + i < H) o[(uint64_t)a * H + r0 + 4 * q + i] = c[i];
}

template <uint32_t kType>
__global__ void mx4_combine(const float *o, const int32_t *ids, const float *w, uint32_t ntok, uint32_t E, uint32_t K,
                            uint32_t H, typename Elem<kType>::T *y, uint64_t stride) {
  const uint64_t i = (uint64_t)blockIdx.x * blockDim.x + threadIdx.x;
  const uint64_t t = i / H;
  const uint32_t c = (uint32_t)(i - t * H);
  if (t >= ntok) return;
  float s = 0.0f;
  for (uint32_t k = 0; k < K; k++)
    if ((uint32_t)ids[t * K + k] < E) s += w[t * K + k] * o[(t * K + k) * H + c];
  y[t * stride + c] = (typename Elem<kType>::T)s;
}

}  // namespace c0ven

using namespace c0ven;

namespace {

void check_experts(const moe_mx4_experts *e, uint32_t ntok) {
  op_require(e != nullptr, "null argument");
  op_require(e->n_embd >= 1 && e->n_embd <= 16384 && e->n_ff >= 1 && e->n_ff <= 16384, "n_embd and n_ff must be 1..16384");
  op_require(e->n_expert >= 1 && e->n_expert <= 512, "n_expert must be 1..512");
  op_require(e->n_used >= 1 && e->n_used <= 16, "n_used must be 1..16");
  op_require(e->swiglu_limit >= 0.0f && e->swiglu_limit < INFINITY, "swiglu_limit must be finite and not negative");
  op_require(ntok <= 16384, "at most 16384 tokens");
  for (const moe_mx4_matrix *m : {&e->gate, &e->up, &e->down}) op_mx4(m);
  op_require(e->gate.rows == e->n_ff && e->gate.cols == e->n_embd && e->up.rows == e->n_ff && e->up.cols == e->n_embd &&
                 e->down.rows == e->n_embd && e->down.cols == e->n_ff,
             "gate and up must be n_ff x n_embd, down n_embd x n_ff");
  op_require(op_float(e->x_type) && op_float(e->y_type), "the element type must be QT_F32, QT_F16 or QT_BF16");
}

// The work buffer's parts: x's rows quantised, h and its rows quantised, the experts' outputs.
struct Work {
  uint64_t xc, xs, h, hc, hs, o, bytes;
  Work(const moe_mx4_experts &e, uint64_t T) {
    uint64_t at = 0;
    const auto part = [&](uint64_t n) {
      const uint64_t was = at;
      at += (n + 255) / 256 * 256;
      return was;
    };
    const uint64_t A = T * e.n_used;
    xc = part(moe_mx4_code_bytes((uint32_t)T, e.n_embd)), xs = part(moe_mx4_scale_bytes((uint32_t)T, e.n_embd));
    h = part(A * e.n_ff * 4);
    hc = part(moe_mx4_code_bytes((uint32_t)A, e.n_ff)), hs = part(moe_mx4_scale_bytes((uint32_t)A, e.n_ff));
    o = part(A * e.n_embd * 4);
    bytes = at;
  }
};

}  // namespace

extern "C" {

MOE_API uint64_t moe_mx4_experts_work_bytes(const moe_mx4_experts *e, uint32_t ntok) {
  uint64_t n = 0;
  (void)op_guarded([&] {
    check_experts(e, ntok);
    n = Work(*e, ntok).bytes;
  });
  return n;
}

MOE_API moe_status moe_mx4_experts_async(const moe_mx4_experts *e, const void *x, uint64_t x_stride, uint32_t ntok,
                                         const int32_t *ids, const float *w, void *y, uint64_t y_stride, void *work,
                                         uint64_t work_bytes, void *stream) {
  return op_guarded([&] {
    check_experts(e, ntok);
    const uint32_t H = e->n_embd, F = e->n_ff, E = e->n_expert, K = e->n_used, A = ntok * K;
    op_rows(x, x_stride, H, e->x_type);
    op_rows(y, y_stride, H, e->y_type);
    op_require(ids && w && op_aligned(ids, 4) && op_aligned(w, 4), "null or misaligned ids or w");
    const Work at(*e, ntok);
    op_work(work, work_bytes, at.bytes);
    if (!ntok) return;
    OnDevice on(e->device);
    uint8_t *b = (uint8_t *)work;
    mx4_quantize_launch(e->x_type, x, x_stride, moe_mx4_matrix{b + at.xc, b + at.xs, ntok, H}, stream);
    op_launch(mx4_gate_up, (uint64_t)A * ((F + 15) / 16), 64, stream, (const uint8_t *)(b + at.xc),
              (const uint8_t *)(b + at.xs), (const uint8_t *)e->gate.codes, (const uint8_t *)e->gate.scales,
              (const uint8_t *)e->up.codes, (const uint8_t *)e->up.scales, ids, E, K, H, F, e->swiglu_limit,
              (float *)(b + at.h));
    mx4_quantize_launch(QT_F32, b + at.h, F, moe_mx4_matrix{b + at.hc, b + at.hs, A, F}, stream);
    op_launch(mx4_down, (uint64_t)A * ((H + 15) / 16), 64, stream, (const uint8_t *)(b + at.hc),
              (const uint8_t *)(b + at.hs), (const uint8_t *)e->down.codes, (const uint8_t *)e->down.scales, ids, E, H, F,
              (float *)(b + at.o));
    const uint64_t n = ((uint64_t)ntok * H + 255) / 256;
    const auto run = [&](auto kernel, auto *p) {
      op_launch(kernel, n, 256, stream, (const float *)(b + at.o), ids, w, ntok, E, K, H, p, y_stride);
    };
    if (e->y_type == QT_F32) run(mx4_combine<QT_F32>, (float *)y);
    if (e->y_type == QT_F16) run(mx4_combine<QT_F16>, (_Float16 *)y);
    if (e->y_type == QT_BF16) run(mx4_combine<QT_BF16>, (__bf16 *)y);
  });
}

}  // extern "C"
