// Routing of logits to experts (moe_route_async).
#include "device_math.h"
#include "mx4.h"
#include "ops.h"

namespace c0ven {

constexpr int kPer = 8;  // experts a lane holds: e = lane + 64 i

__device__ __forceinline__ double wave_max_d(double v) {
  for (int o = 32; o > 0; o >>= 1) v = fmax(v, __shfl_xor(v, o, 64));
  return v;
}

// The largest v of the wave, the lower id first among equals: (v, id) in every lane.
__device__ __forceinline__ void wave_best(double &v, uint32_t &id) {
  for (int o = 32; o > 0; o >>= 1) {
    const double ov = __shfl_xor(v, o, 64);
    const uint32_t oi = __shfl_xor(id, o, 64);
    if (ov > v || (ov == v && oi < id)) v = ov, id = oi;
  }
}

struct RouteArgs {
  uint32_t E, K, groups, kept, best, renorm, sigmoid;
  float scale;
};

// One wave a token, all in fp64.
template <uint32_t kType>
__global__ void __launch_bounds__(256) moe_route(RouteArgs a, const typename Elem<kType>::T *logits, uint64_t stride,
                                                 const float *bias, uint32_t ntok, int32_t *ids, float *w, uint32_t *load) {
  __shared__ double worth_of[4][64];
  const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const uint32_t t = blockIdx.x * 4 + wave;
  const bool on = t < ntok;
  const double kNone = -INFINITY;
  double x[kPer], s[kPer], key[kPer];
  double top = kNone;
#pragma unroll
  for (int i = 0; i < kPer; i++) {
    const uint32_t e = lane + 64 * i;
    const double v = on && e < a.E ? (double)(float)logits[t * stride + e] : kNone;
    x[i] = v > kNone ? v : kNone;
    top = fmax(top, x[i]);
  }
  top = wave_max_d(top);
  double sum = 0.0;
#pragma unroll
  for (int i = 0; i < kPer; i++) {
    s[i] = x[i] == kNone ? 0.0 : a.sigmoid ? 1.0 / (1.0 + exp(-x[i])) : x[i] == top ? 1.0 : exp(x[i] - top);
    sum += s[i];
  }
  if (!a.sigmoid) {
    sum = wave_sum_d(sum);
#pragma unroll
    for (int i = 0; i < kPer; i++) s[i] = sum > 0.0 ? s[i] / sum : 0.0;
  }
#pragma unroll
  for (int i = 0; i < kPer; i++) {
    const uint32_t e = lane + 64 * i;
    key[i] = x[i];
    if (bias && e < a.E) {
      const float b = bias[e];
      key[i] = x[i] > kNone && b > -INFINITY ? s[i] + (double)b : kNone;
    } else if (a.groups > 1 && a.best > 1) {
      key[i] = x[i] > kNone ? s[i] : kNone;
    }
  }
  if (a.groups > 1) {
    const uint32_t n = a.E / a.groups;
    for (uint32_t g = 0; g < a.groups; g++) {  // (all waves go through the barriers together)
      double b1 = kNone, b2 = kNone;
      uint32_t i1 = ~0u, i2 = ~0u;
#pragma unroll
      for (int i = 0; i < kPer; i++) {
        const uint32_t e = lane + 64 * i;
        if (e / n == g && e < a.E && (key[i] > b1 || i1 == ~0u)) b1 = key[i], i1 = e;
      }
      wave_best(b1, i1);
#pragma unroll
      for (int i = 0; i < kPer; i++) {
        const uint32_t e = lane + 64 * i;
        if (e / n == g && e < a.E && e != i1 && (key[i] > b2 || i2 == ~0u)) b2 = key[i], i2 = e;
      }
      wave_best(b2, i2);
      if (lane == 0) worth_of[wave][g] = a.best > 1 && b2 > kNone ? b1 + b2 : b1;
    }
    __syncthreads();
    const double mine = lane < a.groups ? worth_of[wave][lane] : kNone;
    uint32_t place = 0;
    for (uint32_t g = 0; g < a.groups; g++) {
      const double o = worth_of[wave][g];
      place += o > mine || (o == mine && g < lane);
    }
    const uint64_t stays = __ballot(lane < a.groups && place < a.kept);
#pragma unroll
    for (int i = 0; i < kPer; i++) {
      const uint32_t e = lane + 64 * i;
      if (e >= a.E || !(stays >> (e / n) & 1)) key[i] = kNone;
    }
  }
  float mine = 0.0f;
  int32_t my_id = -1;
  for (uint32_t k = 0; k < a.K; k++) {
    double b = kNone;
    uint32_t id = ~0u;
#pragma unroll
    for (int i = 0; i < kPer; i++)
      if (key[i] > b) b = key[i], id = lane + 64 * i;
    wave_best(b, id);
    float v = 0.0f;
#pragma unroll
    for (int i = 0; i < kPer; i++)
      if (id == lane + 64 * i) v = (float)s[i], key[i] = kNone;
    v = __shfl(v, id == ~0u ? 0 : (int)(id & 63), 64);
    if (lane == k) mine = id == ~0u ? 0.0f : v, my_id = (int32_t)id;
  }
  float total = 0.0f;
  for (uint32_t k = 0; k < a.K; k++) total += __shfl(mine, (int)k, 64);
  if (on && lane < a.K) {
    ids[(uint64_t)t * a.K + lane] = my_id;
    w[(uint64_t)t * a.K + lane] = (a.renorm ? mine / fmaxf(total, 1e-20f) : mine) * a.scale;
    if (load && my_id >= 0) atomicAdd(load + my_id, 1u);
  }
}

__global__ void route_clear(uint32_t *load, uint32_t n) {
  if (threadIdx.x < n) load[threadIdx.x] = 0;
}

}  // namespace c0ven

using namespace c0ven;

extern "C" MOE_API moe_status moe_route_async(const moe_route_config *cfg, const void *logits, uint64_t stride,
                                              const float *bias, uint32_t ntok, int32_t *ids, float *w, uint32_t *load,
                                              void *stream) {
  return op_guarded([&] {
    op_require(cfg != nullptr, "null argument");
    const moe_route_config &c = *cfg;
    op_require(c.n_expert >= 1 && c.n_expert <= 512, "n_expert must be 1..512");
    op_require(c.n_used >= 1 && c.n_used <= 16 && c.n_used <= c.n_expert, "n_used must be 1..16 and at most n_expert");
    op_require(c.score == MOE_SCORE_SOFTMAX || c.score == MOE_SCORE_SIGMOID, "unknown score");
    op_require(c.scale >= 0.0f && c.scale < INFINITY, "scale must be finite and not negative");
    op_require(ntok <= 1u << 24, "at most 2^24 tokens");
    if (c.n_group > 1) {
      op_require(c.n_group <= 64 && c.n_expert % c.n_group == 0, "n_group must divide n_expert and be at most 64");
      op_require(c.top_group >= 1 && c.top_group <= c.n_group, "top_group must be 1..n_group");
      op_require(c.group_top == 1 || c.group_top == 2, "group_top must be 1 or 2");
      op_require(c.n_used <= c.n_expert / c.n_group * c.top_group, "n_used exceeds the kept groups' experts");
    }
    op_rows(logits, stride, c.n_expert, c.type);
    op_require(ids && w && op_aligned(ids, 4) && op_aligned(w, 4) && op_aligned(bias, 4) && op_aligned(load, 4),
               "null or misaligned ids, w, bias or load");
    const RouteArgs a{c.n_expert, c.n_used, c.n_group, c.top_group, c.group_top, c.renorm, c.score == MOE_SCORE_SIGMOID,
                      c.scale == 0.0f ? 1.0f : c.scale};
    OnDevice on(c.device);
    if (load) op_launch(route_clear, 1, 512, stream, load, c.n_expert);
    const uint64_t n = (ntok + 3) / 4;
    const auto run = [&](auto kernel, auto *p) { op_launch(kernel, n, 256, stream, a, p, stride, bias, ntok, ids, w, load); };
    if (c.type == QT_F32) run(moe_route<QT_F32>, (const float *)logits);
    if (c.type == QT_F16) run(moe_route<QT_F16>, (const _Float16 *)logits);
    if (c.type == QT_BF16) run(moe_route<QT_BF16>, (const __bf16 *)logits);
  });
}
