// Routing of logits to experts (moe_route_async).
//
// A wave takes a token, then the next that no wave has: its experts lie over the lanes in runs of kPer neighbours. The k
// largest come from a threshold (the k-th largest of the lanes' largest, found bit by bit with ballots: at least k values
// reach it) and the ranking of what reaches it, usually little more than k.
//
// Where the order is that of the logits (no bias, a group's worth from one value) it is exact in fp32 and only the chosen
// need an exponential. Otherwise the order is that of s + bias in fp64: it is formed in fp32 within a bound, and where two
// neighbours of the order (the k-th and the next among them), or the last group kept and the next, are nearer than their
// bounds, the wave does that token again in fp64 (exact_token). Equal logits under equal biases need no bound: their order
// is by id either way.
//
// Bound by memory (the logits read once) where tokens are many, by the launch where they are few. 16384 x 512 fp32, top
// 10: see the figures at moe_route.
#include "device_math.h"
#include "mx4.h"
#include "ops.h"

#include <algorithm>
#include <type_traits>

namespace c0ven {

struct RouteArgs {
  uint32_t E, K, groups, kept, best, renorm, sigmoid;
  float scale;
};

// A token's scratch in LDS, a wave's own.
struct RouteScratch {
  union {
    float v[512];       // the selection values, for the groups
    uint2 cand[64];     // the candidates
  };
};

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
__device__ __forceinline__ float lane_f32(float v, uint32_t l) {
  return __uint_as_float(readlane_u32(__float_as_uint(v), (int)l));
}
__device__ __forceinline__ float wave_sum_f32(float v) {
  v += __uint_as_float(dpp_u32<kDppXor1>(__float_as_uint(v)));
  v += __uint_as_float(dpp_u32<kDppXor2>(__float_as_uint(v)));
  v += __uint_as_float(dpp_u32<kDppHalfMirror>(__float_as_uint(v)));
  v += __uint_as_float(dpp_u32<kDppMirror>(__float_as_uint(v)));
  return (lane_f32(v, 0) + lane_f32(v, 16)) + (lane_f32(v, 32) + lane_f32(v, 48));
}
__device__ __forceinline__ void lds_done() {  // this wave's LDS accesses
  __builtin_amdgcn_s_waitcnt(0xc07f);
  __builtin_amdgcn_wave_barrier();
}

struct Ranked {
  uint32_t id;
  float s;
};
// A token in fp64 throughout: lane r < K receives rank r's id (~0 for none) and score.
template <uint32_t kType, int kPer>
__device__ __noinline__ Ranked exact_token(RouteArgs a, const typename Elem<kType>::T *row, const float *bias) {
  uint32_t my_id = ~0u;
  float my_s = 0.0f;
  const uint32_t lane = threadIdx.x & 63, e0 = lane * kPer;
  const double kNone = -INFINITY;
  double x[kPer], s[kPer], key[kPer], top = kNone, sum = 0.0;
#pragma unroll
  for (int i = 0; i < kPer; i++) {
    const double v = e0 + i < a.E ? (double)(float)row[e0 + i] : kNone;
    x[i] = v > kNone ? v : kNone;  // (no NaN)
    top = fmax(top, x[i]);
  }
  top = wave_max_d(top);
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
    const float b = bias && e0 + i < a.E ? bias[e0 + i] : 0.0f;
    key[i] = x[i] > kNone && b > -INFINITY ? s[i] + (double)b : kNone;
  }
  if (a.groups > 1) {
    const uint32_t n = a.E / a.groups;
    double mine = kNone;  // lane g: group g's worth
    for (uint32_t g = 0; g < a.groups; g++) {
      double b1 = kNone, b2 = kNone;
      uint32_t i1 = ~0u, i2 = ~0u;
#pragma unroll
      for (int i = 0; i < kPer; i++)
        if (e0 + i < a.E && (e0 + i) / n == g && key[i] > b1) b1 = key[i], i1 = e0 + i;
      wave_best(b1, i1);
#pragma unroll
      for (int i = 0; i < kPer; i++)
        if (e0 + i < a.E && (e0 + i) / n == g && e0 + i != i1 && key[i] > b2) b2 = key[i], i2 = e0 + i;
      wave_best(b2, i2);
      if (lane == g) mine = a.best > 1 && b2 > kNone ? b1 + b2 : b1;
    }
    uint32_t place = 0;
    for (uint32_t g = 0; g < a.groups; g++) {
      const double o = __shfl(mine, (int)g, 64);
      place += o > mine || (o == mine && g < lane);
    }
    const uint64_t stays = __ballot(lane < a.groups && place < a.kept);
#pragma unroll
    for (int i = 0; i < kPer; i++)
      if (e0 + i >= a.E || !(stays >> ((e0 + i) / n) & 1)) key[i] = kNone;
  }
  for (uint32_t k = 0; k < a.K; k++) {
    double b = kNone;
    uint32_t id = ~0u;
#pragma unroll
    for (int i = 0; i < kPer; i++)
      if (key[i] > b) b = key[i], id = e0 + i;
    wave_best(b, id);
    float v = 0.0f;
#pragma unroll
    for (int i = 0; i < kPer; i++)
      if (id == e0 + i) v = (float)s[i], key[i] = kNone;
    v = __shfl(v, id == ~0u ? 0 : (int)(id / kPer), 64);
    if (lane == k) my_id = id, my_s = id == ~0u ? 0.0f : v;
  }
  return Ranked{my_id, my_s};
}

// The n largest keys of the wave (0: no key), the lower id first among equals: lane r < n receives the r-th one's key and
// id (key 0 where there are fewer).
template <int kPer>
__device__ __forceinline__ void select_ranks(const uint32_t (&key)[kPer], uint32_t n, RouteScratch &lds, uint32_t &my_key,
                                             uint32_t &my_id) {
  const uint32_t lane = threadIdx.x & 63, e0 = lane * kPer;
  uint32_t m = key[0];
#pragma unroll
  for (int i = 1; i < kPer; i++) m = max(m, key[i]);
  uint32_t tau = 0;
  for (int b = 31; b >= 0; b--) {
    const uint32_t c = tau | (1u << b);
    if ((uint32_t)__popcll(__ballot(m >= c)) >= n) tau = c;
  }
  tau = max(tau, 1u);
  uint32_t cnt = 0, pos = 0, total = 0;  // this lane's candidates, those of the lanes below, all
#pragma unroll
  for (int i = 0; i < kPer; i++) cnt += key[i] >= tau ? 1u : 0u;
#pragma unroll
  for (int b = 0; b < 4; b++) {
    const uint64_t bal = __ballot((cnt >> b) & 1u);
    pos += __builtin_amdgcn_mbcnt_hi((uint32_t)(bal >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)bal, 0u)) << b;
    total += (uint32_t)__popcll(bal) << b;
  }
  if (total <= 64) {
#pragma unroll
    for (int i = 0; i < kPer; i++)
      if (key[i] >= tau) lds.cand[pos++] = make_uint2(key[i], e0 + i);
    lds_done();
    const uint2 me = lane < total ? lds.cand[lane] : make_uint2(0u, 0u);
    lds_done();
    uint32_t rank = 0;
    for (uint32_t i = 0; i < total; i++) {
      const uint32_t ok = readlane_u32(me.x, (int)i), oi = readlane_u32(me.y, (int)i);
      rank += (ok > me.x) | ((ok == me.x) & (oi < me.y));
    }
    const int to = 4 * (int)(lane < total ? rank : lane);  // a permutation of the lanes
    my_key = (uint32_t)__builtin_amdgcn_ds_permute(to, (int)me.x);
    my_id = (uint32_t)__builtin_amdgcn_ds_permute(to, (int)me.y);
    if (lane >= total) my_key = 0u;
    return;
  }
  // (Many equal values.) One after the other: the largest, its lowest lane, that lane's first one.
  uint32_t gone = 0;
  my_key = 0u, my_id = 0u;
  for (uint32_t k = 0; k < n; k++) {
    uint32_t b = 0, at = 0;
#pragma unroll
    for (int i = kPer - 1; i >= 0; i--)
      if (!(gone >> i & 1) && key[i] >= b) b = key[i], at = i;
    const uint32_t top = wave_max_u32(b);
    if (!top) break;
    const uint32_t who = (uint32_t)__ffsll(__ballot(b == top)) - 1;
    if (lane == who) gone |= 1u << at;
    const uint32_t id = who * kPer + readlane_u32(at, (int)who);
    if (lane == k) my_key = top, my_id = id;
  }
}

// kScores: the order is that of s + bias. Tokens go round the grid's waves; load (or null) is counted in LDS and added at
// the end, or stored where one work-group does it all.
template <uint32_t kType, bool kScores, int kPer>
__global__ void __launch_bounds__(512) moe_route(RouteArgs a, const typename Elem<kType>::T *logits, uint64_t stride,
                                                 const float *bias, uint32_t ntok, int32_t *ids, float *w, uint32_t *load) {
  extern __shared__ __align__(16) uint8_t dynamic[];
  uint32_t *count = (uint32_t *)dynamic;  // 512
  RouteScratch *all = (RouteScratch *)(count + 512);
  const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6, waves = blockDim.x / 64, e0 = lane * kPer;
  RouteScratch &lds = all[wave];
  if (load) {
    for (uint32_t e = threadIdx.x; e < a.E; e += blockDim.x) count[e] = 0;
    __syncthreads();
  }
  const uint32_t n = a.groups > 1 ? a.E / a.groups : a.E;
  uint32_t group[kPer];
#pragma unroll
  for (int i = 0; i < kPer; i++) group[i] = (e0 + i) / n;
  for (uint32_t t = blockIdx.x * waves + wave; t < ntok; t += gridDim.x * waves) {
    const typename Elem<kType>::T *row = logits + (uint64_t)t * stride;
    float x[kPer], s[kPer], v[kPer];
    if constexpr (kPer == 8) {
      load8<kType>(row, e0, a.E, x);
    } else {
#pragma unroll
      for (int i = 0; i < kPer; i++) x[i] = e0 + i < a.E ? (float)row[e0 + i] : 0.0f;
    }
#pragma unroll
    for (int i = 0; i < kPer; i++) x[i] = e0 + i < a.E && x[i] > -INFINITY ? x[i] : -INFINITY;
    float top = x[0], sum = 0.0f;
#pragma unroll
    for (int i = 1; i < kPer; i++) top = fmaxf(top, x[i]);
    top = key_float(wave_max_u32(float_key(top)));
    if (!a.sigmoid && (kScores || !a.renorm)) {
#pragma unroll
      for (int i = 0; i < kPer; i++) {
        s[i] = x[i] == -INFINITY ? 0.0f : x[i] == top ? 1.0f : exp_f32(x[i] - top);
        sum += s[i];
      }
      sum = wave_sum_f32(sum);
    }
#pragma unroll
    for (int i = 0; i < kPer; i++) {
      if (kScores) {
        const float b = bias && e0 + i < a.E ? bias[e0 + i] : 0.0f;
        const float p = a.sigmoid ? 1.0f / (1.0f + exp_f32(-x[i])) : s[i] / sum;
        v[i] = x[i] > -INFINITY && b > -INFINITY ? p + b : -INFINITY;
      } else {
        v[i] = x[i];
      }
    }
    bool open = false;  // the order is not certain
    // A score's bound: a few units of its own for the exponential, the quotient and a softmax's sum, and |x - top| of
    // them for the difference, of which e^(x - top) |x - top| <= 0.37 stays: within 2^-20 of the largest score.
    const float off_s = (a.sigmoid ? 1.0f : 1.0f / sum) * 0x1p-20f + 0x1p-120f;
    uint64_t stays = ~0ull;
    if (a.groups > 1) {
      // Lane g goes through group g's values, from a place of its own on, so that the lanes' banks differ.
#pragma unroll
      for (int i = 0; i < kPer; i++)
        if (e0 + i < a.E) lds.v[e0 + i] = v[i];
      lds_done();
      float b1 = -INFINITY, b2 = -INFINITY;
      if (lane < a.groups)
        for (uint32_t j = 0, at = lane % n; j < n; j++, at = at + 1 == n ? 0 : at + 1) {
          const float o = lds.v[lane * n + at];
          b2 = o > b1 ? b1 : fmaxf(b2, o), b1 = fmaxf(b1, o);
        }
      lds_done();
      const float mine = a.best > 1 && b2 > -INFINITY ? b1 + b2 : b1;
      uint32_t place = 0;
      for (uint32_t g = 0; g < a.groups; g++) {
        const float o = lane_f32(mine, g);
        place += o > mine || (o == mine && g < lane);
      }
      stays = __ballot(lane < a.groups && place < a.kept);
      if (kScores && a.kept < a.groups) {
        const uint32_t in = (uint32_t)__ffsll(__ballot(lane < a.groups && place == a.kept - 1)) - 1;
        const uint32_t out = (uint32_t)__ffsll(__ballot(lane < a.groups && place == a.kept)) - 1;
        const float wi = lane_f32(mine, in), wo = lane_f32(mine, out);
        // Four scores, and the roundings of their sums.
        if (wo > -INFINITY) open = !(wi - wo > 4.0f * off_s + 0x1p-20f * (fabsf(wi) + fabsf(wo)));
      }
    }
    uint32_t key[kPer];
#pragma unroll
    for (int i = 0; i < kPer; i++)
      key[i] = v[i] > -INFINITY && (a.groups <= 1 || (stays >> group[i] & 1)) ? float_key(v[i]) : 0u;
    uint32_t my_key, my_id;
    select_ranks<kPer>(key, kScores ? a.K + 1 : a.K, lds, my_key, my_id);
    const bool mine = my_key != 0 && lane <= a.K;
    float my_x = mine ? (float)row[my_id] : 0.0f, my_s = 0.0f;
    if (kScores) {
      const float my_b = mine && bias ? bias[my_id] : 0.0f;
      my_s = a.sigmoid ? 1.0f / (1.0f + exp_f32(-my_x)) : (my_x == top ? 1.0f : exp_f32(my_x - top)) / sum;
      if (!mine) my_s = 0.0f;
      // Rank r against rank r + 1 (any later one's value is no larger, and its bound is the same).
      const float my_v = key_float(my_key);
      const uint32_t next = (lane + 1) & 63;
      const uint32_t nk = __shfl(my_key, next, 64);
      const float nx = __shfl(my_x, next, 64), nb = __shfl(my_b, next, 64);
      const float nv = key_float(nk);
      const bool equal = nx == my_x && nb == my_b;
      const float off = 2.0f * off_s + 0x1p-22f * (fabsf(my_v) + fabsf(nv));
      open |= __any(lane < a.K && mine && nk != 0 && !equal && !(my_v - nv > off));
    } else {
      if (a.sigmoid)
        my_s = 1.0f / (1.0f + exp_f32(-my_x));
      else  // with renorm the common factor drops out: relative to the first chosen
        my_s = a.renorm ? (my_x == lane_f32(my_x, 0) ? 1.0f : exp_f32(my_x - lane_f32(my_x, 0)))
                        : (my_x == top ? 1.0f : exp_f32(my_x - top)) / sum;
    }
    if (kScores && open) {
      const Ranked r = exact_token<kType, kPer>(a, row, bias);
      my_id = r.id, my_s = r.s, my_key = r.id != ~0u;
    }
    if (!(my_key != 0 && lane < a.K)) my_s = 0.0f;
    float total = 0.0f;
    for (uint32_t k = 0; k < a.K; k++) total += lane_f32(my_s, k);
    if (lane < a.K) {
      const uint64_t at = (uint64_t)t * a.K + lane;
      ids[at] = my_key ? (int32_t)my_id : -1;
      w[at] = (a.renorm ? my_s / fmaxf(total, 1e-20f) : my_s) * a.scale;
      if (load && my_key) atomicAdd(count + my_id, 1u);
    }
  }
  if (load) {
    __syncthreads();
    for (uint32_t e = threadIdx.x; e < a.E; e += blockDim.x) {
      if (gridDim.x == 1)
        load[e] = count[e];
      else if (count[e])
        atomicAdd(load + e, count[e]);
    }
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
    if (!ntok && !load) return;
    OnDevice on(c.device);
    // Up to eight tokens are one work-group's, which stores load; more are dealt to at most four waves a SIMD.
    const uint32_t waves = std::min(std::max(ntok, 1u), 8u);
    const uint32_t blocks = (uint32_t)std::min<uint64_t>((ntok + waves - 1) / waves, 512);
    if (load && blocks != 1) op_launch(route_clear, 1, 512, stream, load, c.n_expert);
    const bool scores = bias || (c.n_group > 1 && c.group_top > 1);
    const auto run = [&](auto kernel, auto *p) {
      op_launch_lds(kernel, blocks, 64 * waves, 2048 + waves * (uint32_t)sizeof(RouteScratch), stream, a, p, stride, bias, ntok,
                    ids, w, load);
    };
    const auto typed = [&](auto type, auto *p) {
      constexpr uint32_t kType = decltype(type)::value;
      if (c.n_expert <= 64) return scores ? run(moe_route<kType, true, 1>, p) : run(moe_route<kType, false, 1>, p);
      if (c.n_expert <= 128) return scores ? run(moe_route<kType, true, 2>, p) : run(moe_route<kType, false, 2>, p);
      if (c.n_expert <= 256) return scores ? run(moe_route<kType, true, 4>, p) : run(moe_route<kType, false, 4>, p);
      return scores ? run(moe_route<kType, true, 8>, p) : run(moe_route<kType, false, 8>, p);
    };
    if (c.type == QT_F32) typed(std::integral_constant<uint32_t, QT_F32>(), (const float *)logits);
    if (c.type == QT_F16) typed(std::integral_constant<uint32_t, QT_F16>(), (const _Float16 *)logits);
    if (c.type == QT_BF16) typed(std::integral_constant<uint32_t, QT_BF16>(), (const __bf16 *)logits);
  });
}
