// Routing of logits to experts (moe_route_async).
//
// A wave takes a token, then the next that no wave has: its experts lie over the lanes in runs of kPer neighbours. The k
// largest come from a threshold (the k-th largest of the lanes' largest, found bit by bit with ballots: at least k values
// reach it) and the ranking of what reaches it, usually little more than k.
//
// Where the order is that of the logits (no bias, a group's worth from one value) it is exact in fp32 and only the chosen
// need an exponential. Otherwise the order is that of s + bias in fp64: it is formed in fp32 within a bound, and where two
// neighbours of the order (the k-th and the next among them), or a group and the border between those kept and the others, are
// nearer than their bounds, the wave decides that in fp64: among the candidates, or among all where too many are near. Equal
// logits under equal biases need no bound: their order is by id either way.
//
// Bound by the launch where tokens are few (one of 512 experts, top 10: 4.4 us), else by the instructions of a token: 16384 x
// 512 fp32, top 10, 293 vector and 219 scalar ones, 13.6 us (2.5 TB/s; the logits alone are 6.8 us at 5.1) and 3.8 for the load;
// with biases 576 and 294 on half the waves (fp64's registers), 36 us and 4.5. 999 x 256 bf16 with biases and groups 10.4 and
// 2.9 us (in a graph of such calls 7.0 and 2.4): one token a wave, its latency, and some tokens' fp64.
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

// The same values as ones of their own to the compiler, so that what is computed from them stays where it is used: it moved
// some 30 conditions before the tokens' loop and kept them, two scalars each, in lanes of a register (999 x 256 with groups
// 9.6 us, 7.1 with this).
__device__ __forceinline__ RouteArgs apart(RouteArgs a) {
  asm volatile("" : "+s"(a.E), "+s"(a.K), "+s"(a.groups), "+s"(a.kept), "+s"(a.best), "+s"(a.sigmoid));
  return a;
}

// A token's scratch in LDS, a wave's own.
struct RouteScratch {
  union {
    float v[512];       // the selection values, for the groups
    float2 best[64];    // a lane's largest two
    double d[512];      // the same in fp64
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
template <int kCtrl>
__device__ __forceinline__ float dpp_f32(float v) {
  return __uint_as_float(dpp_u32<kCtrl>(__float_as_uint(v)));
}
__device__ __forceinline__ float wave_sum_f32(float v) {
  v += dpp_f32<kDppXor1>(v);
  v += dpp_f32<kDppXor2>(v);
  v += dpp_f32<kDppHalfMirror>(v);
  v += dpp_f32<kDppMirror>(v);
  return (lane_f32(v, 0) + lane_f32(v, 16)) + (lane_f32(v, 32) + lane_f32(v, 48));
}
__device__ __forceinline__ void lds_done() {  // this wave's LDS accesses
  __builtin_amdgcn_s_waitcnt(0xc07f);
  __builtin_amdgcn_wave_barrier();
}

// Chosen scores are held 2^70 times as large where they may be tiny: over the renormaliser's floor of 1e-20 the weights are
// numbers of fp32 down to scores of 2^-192. A token whose order is the scores' is left to fp64 where a chosen one is below
// kTiny (scores lifted in fp32 there too: 999 x 256 with groups 9.6 us, 9.4).
constexpr float kLift = 0x1p70f;
constexpr float kTiny = 0x1p-60f;
// exp(z) as exp_f32, or where far (z < -80) kLift times it.
__device__ __forceinline__ float exp_lifted(float z, bool far) {
  z = z < -200.0f ? -200.0f : z > 89.0f ? 89.0f : z;
  const float hi = z * 1.4426950216e+0f;
  const float lo = __builtin_fmaf(z, 1.9259629911e-8f, __builtin_fmaf(z, 1.4426950216e+0f, -hi));
  return __builtin_amdgcn_exp2f(far ? hi + 70.0f : hi) * __builtin_fmaf(lo, 0.69314718f, 1.0f);
}
// kLift times a sigmoid, and times a softmax's score of the largest logit top and the sum of e^(x - top).
__device__ __forceinline__ float lifted_sigmoid(float x) {
  const bool far = x < -80.0f;  // (1 + e^x is 1)
  const float e = exp_lifted(far ? x : -x, far);
  return far ? e : kLift / (1.0f + e);
}
__device__ __forceinline__ float lifted_softmax(float x, float top, float sum) {
  const bool far = x - top < -80.0f;
  const float e = exp_lifted(x - top, far);
  return (x == top ? kLift : far ? e : kLift * e) / sum;
}

// The scores in fp64 of the lanes' logits (minus infinity: no score): a softmax's largest logit and sum (1 for a sigmoid).
struct Exact {
  double top = -INFINITY, sum = 1.0;

  template <int kPer>
  __device__ __forceinline__ Exact(const RouteArgs &a, const float (&x)[kPer]) {
    if (a.sigmoid) return;
    float m = x[0];
#pragma unroll
    for (int i = 1; i < kPer; i++) m = fmaxf(m, x[i]);
    top = (double)key_float(wave_max_u32(float_key(m)));
    sum = 0.0;
#pragma unroll
    for (int i = 0; i < kPer; i++) sum += part(a, x[i]);
    sum = wave_sum_f64(sum);
  }
  __device__ __forceinline__ double part(const RouteArgs &a, float xf) const {
    const double x = (double)xf;
    return xf == -INFINITY ? 0.0 : a.sigmoid ? 1.0 / (1.0 + exp(-x)) : x == top ? 1.0 : exp(x - top);
  }
  __device__ __forceinline__ double score(const RouteArgs &a, float x) const { return sum > 0.0 ? part(a, x) / sum : 0.0; }
  // The values that select, into LDS (minus infinity: not to be selected).
  template <int kPer>
  __device__ __forceinline__ void keys(const RouteArgs &a, const float (&x)[kPer], const float (&b)[kPer], double *d) const {
    const uint32_t e0 = (threadIdx.x & 63) * kPer;
#pragma unroll
    for (int i = 0; i < kPer; i++)
      if (e0 + i < a.E) d[e0 + i] = x[i] > -INFINITY && b[i] > -INFINITY ? score(a, x[i]) + (double)b[i] : -INFINITY;
    lds_done();
  }
};

// The groups that stay, decided on the values in d.
__device__ __forceinline__ uint64_t exact_groups(const RouteArgs &a, const double *d) {
  const uint32_t lane = threadIdx.x & 63, n = a.E / a.groups;
  double b1 = -INFINITY, b2 = -INFINITY;
  if (lane < a.groups)
    for (uint32_t j = 0; j < n; j++) {
      const double o = d[lane * n + j];
      b2 = o > b1 ? b1 : fmax(b2, o), b1 = fmax(b1, o);
    }
  lds_done();
  const double mine = a.best > 1 && b2 > -INFINITY ? b1 + b2 : b1;
  uint32_t place = 0;
  for (uint32_t g = 0; g < a.groups; g++) {
    const double o = readlane_f64(mine, (int)g);
    place += o > mine || (o == mine && g < lane);
  }
  return __ballot(lane < a.groups && place < a.kept);
}

struct Ranked {
  uint32_t id;  // ~0: none
  float s;      // kLift times its score
};
// The ranks in fp64 among the candidates that lanes 0 .. total - 1 hold (id, logit, bias): lane r receives rank r.
__device__ __forceinline__ Ranked exact_ranks(const RouteArgs &a, const Exact &e, uint32_t total, uint32_t id, float x, float b) {
  const uint32_t lane = threadIdx.x & 63;
  const double s = e.score(a, x), key = s + (double)b;
  uint32_t rank = 0;
  for (uint32_t i = 0; i < total; i++) {
    const double o = readlane_f64(key, (int)i);
    rank += o > key || (o == key && readlane_u32(id, (int)i) < id);
  }
  const int to = 4 * (int)(lane < total ? rank : lane);
  const uint32_t ri = (uint32_t)__builtin_amdgcn_ds_permute(to, (int)id);
  const float rs = __uint_as_float((uint32_t)__builtin_amdgcn_ds_permute(to, (int)__float_as_uint((float)(s * (double)kLift))));
  return lane < total ? Ranked{ri, rs} : Ranked{~0u, 0.0f};
}
// The ranks of the values in d (changed) among the experts of the groups that stay, one after the other.
template <uint32_t kType, int kPer>
__device__ __forceinline__ Ranked exact_all(const RouteArgs &a, const Exact &e, const typename Elem<kType>::T *row,
                                            uint64_t stays, double *d) {
  const uint32_t lane = threadIdx.x & 63, e0 = lane * kPer, n = a.groups > 1 ? a.E / a.groups : a.E;
  Ranked mine{~0u, 0.0f};
  for (uint32_t k = 0; k < a.K; k++) {
    double b = -INFINITY;
    uint32_t id = ~0u;
#pragma unroll 1
    for (int i = 0; i < kPer; i++) {
      if (e0 + i >= a.E) break;
      const double v = d[e0 + i];
      if (v > b && (stays >> ((e0 + i) / n) & 1)) b = v, id = e0 + i;
    }
    wave_best(b, id);
    if (id == ~0u) break;
    if (id / kPer == lane) d[id] = -INFINITY;
    if (lane == k) mine.id = id;
  }
  lds_done();
  if (mine.id != ~0u) mine.s = (float)(e.score(a, (float)row[mine.id]) * (double)kLift);
  return mine;
}

// The n largest keys of the wave (up to kNoKey: none), the lower id first among equals: lane r receives the r-th one's key and
// id (key 0 where there are fewer), for r below the number returned, at least n where there are so many; every other
// expert's key is at most floor.
constexpr uint32_t kNoKey = 0x007fffffu;  // minus infinity's
template <int kPer>
__device__ __forceinline__ uint32_t select_ranks(const uint32_t (&key)[kPer], uint32_t n, RouteScratch &lds, uint32_t &my_key,
                                                 uint32_t &my_id, uint32_t &floor) {
  const uint32_t lane = threadIdx.x & 63, e0 = lane * kPer;
  uint32_t m = key[0];
#pragma unroll
  for (int i = 1; i < kPer; i++) m = max(m, key[i]);
  uint32_t tau = 0;
  for (int b = 31; b >= 0; b--) {
    const uint32_t c = tau | (1u << b);
    const uint32_t reach = (uint32_t)__popcll(__ballot(m >= c));
    if (reach >= n) tau = c;
    if (reach == n) break;  // (no lower bit changes who reaches it)
  }
  floor = tau;
  tau = max(tau, kNoKey + 1);
  uint32_t total = 0;
#pragma unroll
  for (int i = 0; i < kPer; i++) total += (uint32_t)__popcll(__ballot(key[i] >= tau));
  if (total <= 64) {
    uint32_t base = 0;
#pragma unroll
    for (int i = 0; i < kPer; i++) {
      const uint64_t bal = __ballot(key[i] >= tau);
      const uint32_t pos = __builtin_amdgcn_mbcnt_hi((uint32_t)(bal >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)bal, base));
      if (key[i] >= tau) lds.cand[pos] = make_uint2(key[i], e0 + i);
      base += (uint32_t)__popcll(bal);
    }
    lds_done();
    const uint2 me = lane < total ? lds.cand[lane] : make_uint2(0u, 0u);
    lds_done();
    uint32_t rank = 0;
    const uint64_t mine = (uint64_t)me.x << 32 | ~me.y;
    for (uint32_t i = 0; i < total; i++) {
      const uint32_t ok = readlane_u32(me.x, (int)i), oi = readlane_u32(me.y, (int)i);
      rank += ((uint64_t)ok << 32 | ~oi) > mine ? 1u : 0u;
    }
    const int to = 4 * (int)(lane < total ? rank : lane);  // a permutation of the lanes
    my_key = (uint32_t)__builtin_amdgcn_ds_permute(to, (int)me.x);
    my_id = (uint32_t)__builtin_amdgcn_ds_permute(to, (int)me.y);
    if (lane >= total) my_key = 0u;
    return total;
  }
  // (Many equal values.) One after the other: the largest, its lowest lane, that lane's first one.
  uint32_t gone = 0;
  my_key = 0u, my_id = 0u;
  uint32_t k = 0;
  for (; k < n; k++) {
    uint32_t b = 0, at = 0;
#pragma unroll
    for (int i = kPer - 1; i >= 0; i--)
      if (!(gone >> i & 1) && key[i] >= b) b = key[i], at = i;
    const uint32_t top = wave_max_u32(b);
    floor = top;
    if (top <= kNoKey) break;
    const uint32_t who = (uint32_t)__ffsll(__ballot(b == top)) - 1;
    if (lane == who) gone |= 1u << at;
    const uint32_t id = who * kPer + readlane_u32(at, (int)who);
    if (lane == k) my_key = top, my_id = id;
  }
  return k;
}

// A row's kPer values from column c on (0 past cols), in one load where all are there.
template <uint32_t kType, int kPer>
__device__ __forceinline__ void load_run(const typename Elem<kType>::T *row, uint32_t c, uint32_t cols, float (&v)[kPer]) {
  typedef typename Elem<kType>::T T;
  struct __attribute__((packed)) Pack {
    T e[kPer];
  };
#pragma unroll
  for (int j = 0; j < kPer; j++) v[j] = 0.0f;
  if (c + kPer <= cols) {
    const Pack p = *(const Pack *)(row + c);
#pragma unroll
    for (int j = 0; j < kPer; j++) v[j] = (float)p.e[j];
  } else if (c < cols) {
#pragma unroll
    for (uint32_t j = 0; j < kPer - 1; j++)
      if (c + j < cols) v[j] = (float)row[c + j];
  }
}

// kScores: the order is that of s + bias. Tokens go round the grid's waves. load (or null): one work-group counts it; of
// several the first clears it for route_count.
template <uint32_t kType, bool kScores, int kPer>
__global__ void __launch_bounds__(kScores && kPer == 8 ? 512 : 1024) moe_route(RouteArgs a, const typename Elem<kType>::T *logits, uint64_t stride,
                                                 const float *bias, uint32_t ntok, int32_t *ids, float *w, uint32_t *load) {
  extern __shared__ __align__(16) uint8_t dynamic[];
  uint32_t *count = (uint32_t *)dynamic;  // 512
  RouteScratch *all = (RouteScratch *)(count + 512);
  const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6, waves = blockDim.x / 64, e0 = lane * kPer;
  RouteScratch &lds = all[wave];
  const bool counts = load && gridDim.x == 1;
  if (counts) {
    for (uint32_t e = threadIdx.x; e < a.E; e += blockDim.x) count[e] = 0;
    __syncthreads();
  } else if (load && blockIdx.x == 0) {
    for (uint32_t e = threadIdx.x; e < a.E; e += blockDim.x) load[e] = 0;
  }
  const uint32_t step = gridDim.x * waves, n = a.groups > 1 ? a.E / a.groups : a.E;
  // lane r < K: rank r's expert (~0: none) and its score, or kLift times it
  const auto finish = [&](uint32_t t, uint32_t id, float score, bool lifted) {
    if (id == ~0u || lane >= a.K) score = 0.0f;
    float all_s = score;  // the sum of the first sixteen lanes
    all_s += dpp_f32<kDppXor1>(all_s);
    all_s += dpp_f32<kDppXor2>(all_s);
    all_s += dpp_f32<kDppHalfMirror>(all_s);
    all_s += dpp_f32<kDppMirror>(all_s);
    if (lane >= a.K) return;
    const uint64_t at = (uint64_t)t * a.K + lane;
    ids[at] = (int32_t)id;
    w[at] = (a.renorm ? score / fmaxf(all_s, lifted ? 1e-20f * kLift : 1e-20f) : lifted ? score * (1.0f / kLift) : score) * a.scale;
    if (counts && id != ~0u) atomicAdd(count + id, 1u);
  };
  // The tokens whose order fp32 decides, one after the other; at one that it leaves open the loop is left and entered
  // again, so that what only it needs (the next token's logits, the biases) is in no register beside fp64's.
  const uint32_t per_group = ((1u << 20) + n - 1) / n;  // e per_group >> 20 = e / n for e < 512
  // A group of a power of two lanes is compared lane by lane.
  const uint32_t run = a.groups > 1 && n % kPer == 0 && (n / kPer & (n / kPer - 1)) == 0 ? n / kPer : 0;
  uint64_t stays = ~0ull;
  bool decided = false;  // stays, for token t, in fp64
  for (uint32_t t = blockIdx.x * waves + wave; t < ntok;) {
    float b[kPer] = {};
    if (kScores && bias) load_run<QT_F32, kPer>(bias, e0, a.E, b);
    bool open = false, open_groups = false;
    uint32_t my_key, my_id, floor, total;
    float x[kPer], my_x, my_b = 0.0f, off_s = 0.0f;
    for (; t < ntok; t += step) {
      const RouteArgs h = apart(a);  // (the arguments, here)
      uint32_t lanes_of = run;
      asm volatile("" : "+s"(lanes_of));
      const typename Elem<kType>::T *row = logits + (uint64_t)t * stride;
      float s[kPer], v[kPer];
      load_run<kType, kPer>(row, e0, h.E, x);
#pragma unroll
      for (int i = 0; i < kPer; i++) x[i] = x[i] > -INFINITY ? x[i] : -INFINITY;  // (no NaN)
      if (h.E < 64 * kPer) {
#pragma unroll
        for (int i = 0; i < kPer; i++) x[i] = e0 + i < h.E ? x[i] : -INFINITY;
      }
      float top = x[0], sum = 0.0f;
#pragma unroll
      for (int i = 1; i < kPer; i++) top = fmaxf(top, x[i]);
      top = key_float(wave_max_u32(float_key(top)));
      if (!h.sigmoid && (kScores || !h.renorm)) {
#pragma unroll
        for (int i = 0; i < kPer; i++) {
          const float p = exp_f32(x[i] - top);
          s[i] = x[i] == top ? 1.0f : p;
          s[i] = x[i] > -INFINITY ? s[i] : 0.0f;
          sum += s[i];
        }
        sum = wave_sum_f32(sum);
      }
      const float per_sum = h.sigmoid ? 1.0f : __builtin_amdgcn_rcpf(sum);
      if (kScores && h.sigmoid) {
#pragma unroll
        for (int i = 0; i < kPer; i++) s[i] = __builtin_amdgcn_rcpf(1.0f + exp_f32(-x[i]));
      }
#pragma unroll
      for (int i = 0; i < kPer; i++) {
        v[i] = kScores ? s[i] * per_sum + b[i] : x[i];
        if (kScores) v[i] = (x[i] > -INFINITY) & (b[i] > -INFINITY) ? v[i] : -INFINITY;
      }
      // A score's bound: a few units of its own for the exponential, the quotient and a softmax's sum, and |x - top| of
      // them for the difference, of which e^(x - top) |x - top| <= 0.37 stays: within 2^-20 of the largest score.
      off_s = per_sum * 0x1p-20f + 0x1p-120f;
      if (h.groups > 1 && !decided) {
        float b1 = -INFINITY, b2 = -INFINITY;
        uint32_t at = lane;  // this lane's group; of a lanes_of of lanes a group, each has it
        if (lanes_of) {
#pragma unroll
          for (int i = 0; i < kPer; i++) b2 = fmaxf(b2, fminf(b1, v[i])), b1 = fmaxf(b1, v[i]);
          const auto merge = [&](float o1, float o2) { b2 = fmaxf(fminf(b1, o1), fmaxf(b2, o2)), b1 = fmaxf(b1, o1); };
          if (lanes_of > 1) merge(dpp_f32<kDppXor1>(b1), dpp_f32<kDppXor1>(b2));
          if (lanes_of > 2) merge(dpp_f32<kDppXor2>(b1), dpp_f32<kDppXor2>(b2));
          if (lanes_of > 4) merge(dpp_f32<kDppHalfMirror>(b1), dpp_f32<kDppHalfMirror>(b2));
          if (lanes_of > 8) merge(dpp_f32<kDppMirror>(b1), dpp_f32<kDppMirror>(b2));
          if (lanes_of > 16) merge(__shfl_xor(b1, 16, 64), __shfl_xor(b2, 16, 64));
          if (lanes_of > 32) merge(__shfl_xor(b1, 32, 64), __shfl_xor(b2, 32, 64));
          at = e0 / n;
        } else if (n % kPer == 0) {
          // Lane g joins its group's lanes' largest two.
#pragma unroll
          for (int i = 0; i < kPer; i++) b2 = fmaxf(b2, fminf(b1, v[i])), b1 = fmaxf(b1, v[i]);
          lds.best[lane] = make_float2(b1, b2);
          lds_done();
          b1 = b2 = -INFINITY;
          const uint32_t lanes = n / kPer;
          if (lane < h.groups)
            for (uint32_t j = 0; j < lanes; j++) {
              const float2 o = lds.best[lane * lanes + j];
              b2 = fmaxf(fminf(b1, o.x), fmaxf(b2, o.y)), b1 = fmaxf(b1, o.x);
            }
          lds_done();
        } else {
          // Lane g goes through group g's values, from a place of its own on, so that the lanes' banks differ.
#pragma unroll
          for (int i = 0; i < kPer; i++)
            if (e0 + i < h.E) lds.v[e0 + i] = v[i];
          lds_done();
          if (lane < h.groups)
#pragma unroll 8
            for (uint32_t j = 0, k = lane % n; j < n; j++, k = k + 1 == n ? 0 : k + 1) {
              const float o = lds.v[lane * n + k];
              b2 = fmaxf(b2, fminf(b1, o)), b1 = fmaxf(b1, o);
            }
          lds_done();
        }
        const float mine = h.best > 1 && b2 > -INFINITY ? b1 + b2 : b1;
        uint32_t place = 0;
        for (uint32_t g = 0; g < h.groups; g++) {
          const float o = lane_f32(mine, lanes_of ? g * lanes_of : g);
          place += o > mine || (o == mine && g < at);
        }
        const uint64_t keep = __ballot(at < h.groups && place < h.kept);
        stays = keep;
        if (lanes_of > 1) {
          stays = 0;
          for (uint32_t g = 0; g < h.groups; g++) stays |= (keep >> (g * lanes_of) & 1) << g;
        }
        if (kScores && h.kept < h.groups) {
          const uint32_t in = (uint32_t)__ffsll(__ballot(at < h.groups && place == h.kept - 1)) - 1;
          const uint32_t out = (uint32_t)__ffsll(__ballot(at < h.groups && place == h.kept)) - 1;
          const float wi = lane_f32(mine, in), wo = lane_f32(mine, out);
          // Every group against halfway between the last kept and the next: two scores, and their sums' roundings, which are
          // those of the larger value where the two cancel.
          const float half = 0.5f * wi + 0.5f * wo;
          const float off = 2.0f * off_s + 0x1p-20f * (h.best > 1 && b2 > -INFINITY ? fabsf(b1) + fabsf(b2) : fabsf(b1));
          const bool far = place < h.kept ? mine - off > half : mine + off < half;
          open_groups = wo > -INFINITY && __any(at < h.groups && mine > -INFINITY && !far);
          if (open_groups) break;
        }
      }
      uint32_t key[kPer];
#pragma unroll
      for (int i = 0; i < kPer; i++) key[i] = float_key(v[i]);
      if (h.groups > 1) {
#pragma unroll
        for (int i = 0; i < kPer; i++) key[i] = stays >> ((e0 + i) * per_group >> 20) & 1 ? key[i] : 0u;
      }
      // (A few ranks past the last, so that what an open order may move lies among them.)
      total = select_ranks<kPer>(key, kScores ? h.K + 4 : h.K, lds, my_key, my_id, floor);
      const bool mine = my_key != 0 && lane <= h.K;
      my_x = my_key != 0 ? (float)row[my_id] : -INFINITY;
      float my_s;
      if (kScores)
        my_s = h.sigmoid ? 1.0f / (1.0f + exp_f32(-my_x)) : (my_x == top ? 1.0f : exp_f32(my_x - top)) / sum;
      else if (h.sigmoid)
        my_s = lifted_sigmoid(my_x);
      else if (!h.renorm)
        my_s = lifted_softmax(my_x, top, sum);
      else  // with renorm the common factor drops out: relative to the first chosen
        my_s = kLift * (my_x == lane_f32(my_x, 0) ? 1.0f : exp_f32(my_x - lane_f32(my_x, 0)));
      if (kScores) {
        // Rank r against rank r + 1 (any later one's value is no larger, and its bound is the same). Where the last rank's
        // equal is next, with it every expert that is no larger: what is not its equal may be larger in fp64 than both.
        my_b = my_key != 0 && bias ? bias[my_id] : 0.0f;
        const float my_v = key_float(my_key);
        const uint32_t next = (lane + 1) & 63;
        const uint32_t nk = __shfl(my_key, next, 64);
        const float nx = __shfl(my_x, next, 64), nb = __shfl(my_b, next, 64), nv = key_float(nk);
        const float off = 2.0f * off_s + 0x1p-22f * (fabsf(my_v) + fabsf(nv));
        const bool equal = nx == my_x && nb == my_b;
        open = __any(lane < h.K && mine && ((nk != 0 && !equal && !(my_v - nv > off)) || my_s < kTiny));
        if (open) break;
        if (__any(lane == h.K - 1 && mine && nk != 0 && equal)) {
          // (o is near v if v - o <= 2 off_s + 2^-22 (|v| + |o|), so v - o is at most this:)
          const uint32_t last = readlane_u32(my_key, (int)h.K - 1);
          const float lv = key_float(last), lx = lane_f32(my_x, h.K - 1), lb = lane_f32(my_b, h.K - 1);
          const float gap = 2.01f * off_s + 0x1.2p-21f * fabsf(lv);
          const uint32_t low = max(float_key(lv < INFINITY ? lv - gap : lv), kNoKey + 1);
          bool near = false;
#pragma unroll
          for (int i = 0; i < kPer; i++) near |= (key[i] >= low) & (key[i] <= last) & ((x[i] != lx) | (b[i] != lb));
          open = __any(near);
          if (open) break;
        }
      }
      finish(t, mine ? my_id : ~0u, my_s, !kScores);
      decided = false;
    }
    if (!kScores || t >= ntok) break;
    const RouteArgs c = apart(a);
    const Exact e(c, x);
    if (open_groups) {
      e.keys(c, x, b, lds.d);
      stays = exact_groups(c, lds.d);
      decided = true;
      continue;
    }
    // All that may belong to the first K are in the lanes if what is not there is below the K-th by more.
    const float last = lane_f32(key_float(my_key), c.K - 1), rest = key_float(floor);
    Ranked r;
    if (floor <= kNoKey || readlane_u32(my_key, (int)c.K - 1) == 0 ||
        last - rest > 2.0f * off_s + 0x1p-22f * (fabsf(last) + fabsf(rest))) {
      r = exact_ranks(c, e, total, my_id, my_x, my_b);
    } else {
      e.keys(c, x, b, lds.d);
      r = exact_all<kType, kPer>(c, e, logits + (uint64_t)t * stride, stays, lds.d);
    }
    finish(t, r.id, r.s, true);
    decided = false;
    t += step;
  }
  if (counts) {
    __syncthreads();
    for (uint32_t e = threadIdx.x; e < a.E; e += blockDim.x) load[e] = count[e];
  }
}

// How often each expert is among the n ids, into load: stored by one work-group, added by several (load is cleared).
// After the routing, so that the 512 counters see a few work-groups' sums and not each of hundreds (16384 tokens: 4 us
// instead of +12).
constexpr uint32_t kCountIds = 16384;  // a work-group's
__global__ void __launch_bounds__(1024) route_count(const int32_t *ids, uint32_t n, uint32_t E, uint32_t *load) {
  __shared__ uint32_t count[512];
  if (threadIdx.x < 512) count[threadIdx.x] = 0;
  __syncthreads();
  int32_t id[kCountIds / 1024];
#pragma unroll
  for (uint32_t j = 0; j < kCountIds / 1024; j++) {
    const uint32_t i = blockIdx.x * kCountIds + j * 1024 + threadIdx.x;
    id[j] = i < n ? ids[i] : -1;
  }
#pragma unroll
  for (uint32_t j = 0; j < kCountIds / 1024; j++)
    if (id[j] >= 0) atomicAdd(count + id[j], 1u);
  __syncthreads();
  if (threadIdx.x >= E) return;
  if (gridDim.x == 1)
    load[threadIdx.x] = count[threadIdx.x];
  else if (count[threadIdx.x])
    atomicAdd(load + threadIdx.x, count[threadIdx.x]);
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
    op_rows(logits, stride, ntok, c.n_expert, c.type);
    op_require(((ids && w) || !ntok) && op_aligned(ids, 4) && op_aligned(w, 4) && op_aligned(bias, 4) && op_aligned(load, 4),
               "null or misaligned ids, w, bias or load");
    const uint32_t groups = c.top_group < c.n_group ? c.n_group : 1;  // (all of them kept: as none)
    const RouteArgs a{c.n_expert, c.n_used, groups, c.top_group, c.group_top, c.renorm, c.score == MOE_SCORE_SIGMOID,
                      c.scale == 0.0f ? 1.0f : c.scale};
    if (!ntok && !load) return;
    OnDevice on(c.device);
    if (!ntok) return op_launch(route_clear, 1, 512, stream, load, c.n_expert);
    // The order is the scores', also where all groups are kept: logits that are apart may have equal ones in 64 bits.
    const bool scores = bias || (c.n_group > 1 && c.group_top > 1);
    // With load as many tokens as a work-group has waves are one work-group's, which counts (13 tokens of 160 experts with
    // groups 10.6 us, two tokens a wave 17.0; another launch is 2 to 3); more are dealt to as many work-groups as the CUs
    // hold at once, three a CU or, of the scores' larger ones, two (16384 x 512 without a bias with 768 of them 13.3 us, with
    // 512 15.7, with 1024 14.8; with one 41.5, 39.8, 43.6).
    const bool one = load && ntok <= (scores && c.n_expert > 256 ? 8u : 16u);
    const uint32_t waves = std::min(ntok, one ? 16u : 8u), blocks = one ? 1 : std::min((ntok + waves - 1) / waves, scores ? 512u : 768u);
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
    const uint32_t n = ntok * c.n_used;
    if (load && blocks > 1)
      op_launch(route_count, (n + kCountIds - 1) / kCountIds, 1024, stream, (const int32_t *)ids, n, c.n_expert, load);
  });
}
