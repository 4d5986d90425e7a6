// The experts of routed tokens in I8 (moe_i8_experts_async).
//
// Many tokens: the assignments are sorted by expert and cut into MoeTiles; x's rows are quantised; gate and up of a tile are one
// product whose epilogue applies the SwiGLU; the rows of h (fp32: a row's scale needs all of it) are quantised; down follows, its
// values in fp32 by position, and each token's are summed in rank order (in fp32: a value rounded to y's type there would be rounded
// twice). Of 512 experts of 2048 x 512 with a skewed router, 10 a token: 4096 tokens 403 us a call in a row (traced one launch at a time
// 447: gate and up 194, 0.9 POPS with a third of the tiles' rows empty; h quantised 20; down 155, for 0.34 GB of values; their sum 56;
// the sort and x 22), 30 54; 1024 tokens of 8 of 128 experts 144; 301 of 10 of 512 of 2560 x 640 135, where the weights' bytes bound
// it (gate and up 72 us, 4.6 TB/s).
#include "../../include/c0ven_moe_tile.h"
#include "dispatch.h"
#include "experts.h"
#include "i8_api.h"
#include "i8_few.h"
#include "i8_gemm.h"
#include "i8_quant.h"
#include "sort.h"

#include <algorithm>

namespace c0ven {

struct I8Experts {
  const int8_t *gc, *uc, *dc;
  const float *gs, *us, *ds;
  uint32_t E, K, H, F;
  float limit;
};

// expert_swiglu for the epilogue of a tile, a sixth of whose time it was: one reciprocal, good to a unit of the last place, for the
// division's ten instructions. What that loses: on 2^24 normal g the result is off by 5.6e-8 of itself (root of the mean square) and
// 2.6e-7 at most, expert_swiglu's by 4.9e-8 and 2.3e-7, beside the three roundings of g and of u. Below g = -87.3, where the
// reciprocal would be a denormal number, 0 (expert_swiglu from -88.7 on). NaNs and infinities as there: g is a factor of the result.
__device__ __forceinline__ float i8_swiglu(float g, float u, float limit) {
  if (limit > 0.0f) {
    g = g > limit ? limit : g;
    u = u > limit ? limit : u < -limit ? -limit : u;
  }
  const float x = __builtin_amdgcn_fmed3f(-g, -104.0f, 89.0f), hi = x * 1.4426950216e+0f;  // (as exp_f32)
  const float lo = __builtin_fmaf(x, 1.9259629911e-8f, __builtin_fmaf(x, 1.4426950216e+0f, -hi));
  const float e = __builtin_amdgcn_exp2f(hi) * __builtin_fmaf(lo, 0.69314718f, 1.0f);
  return g * __builtin_amdgcn_rcpf(1.0f + e) * u;
}

// The first `slices` work-groups sort (kCount: count their slices' experts), the others quantise x's rows, 16 at a time or (kLong,
// more than 2048 values) one: two launches' work in one (30 tokens 57.7 us, 54.4).
template <uint32_t kX, bool kLong, bool kCount>
__global__ void __launch_bounds__(1024) i8_prepare(const int32_t *ids, uint32_t A, uint32_t E, uint32_t slices, uint32_t *counts,
                                                   SortOut out, const typename Elem<kX>::T *x, uint64_t stride, uint32_t ntok, uint32_t H,
                                                   int8_t *xc, float *xs) {
  if (blockIdx.x >= slices)
    quantize_block<kX, 1024, kLong ? 1024 : 64, kLong ? 2 : 4, false>(blockIdx.x - slices, gridDim.x - slices, x, stride, ntok, H, nullptr,
                                                                      xc, xs);
  else if (kCount)
    count_slice(ids, A, E, kSlice, counts);
  else
    place_slice<true>(ids, A, E, kSlice, 1, nullptr, out);
}

// A tile as scalars (a launch only reads them).
__device__ __forceinline__ MoeTile tile_at(const MoeTile *tiles, uint32_t i) {
  typedef uint32_t __attribute__((ext_vector_type(4))) Four;
  const Four v = *(const __attribute__((address_space(4))) Four *)(uint64_t)(tiles + i);
  return MoeTile{v[0], v[1], v[2], v[3]};
}

// An item: a tile and 64 columns of h (their rows of gate and of up). Writes the positions' rows of h, `pitch` apart: a lane has a
// column of 16 rows, so that a store is of whole lines. A work-group has every gridDim-th item: the next one's tile, ids and first
// two stages are there when it begins (4096 tokens of 10 of 512 experts: 194 us with a work-group an item, 183; down 162 and 150).
template <int TM, bool kLimit>
__global__ void __launch_bounds__(256) i8_gate_up_tiles(I8Experts p, const int8_t *xc, const float *xs, uint32_t ntok,
                                                        const int32_t *order, const MoeTile *tiles, const uint32_t *n_tiles,
                                                        float *h, uint32_t pitch) {
  typedef I8Tile<TM, 2, 2, true, true> Tile;
  constexpr uint32_t kCols = Tile::BN / 2;
  __shared__ typename Tile::X x0;
  __shared__ typename Tile::X x1;
  __shared__ typename Tile::W w0;
  __shared__ typename Tile::W w1;
  __shared__ __align__(16) float sx[2][Tile::BM];
  typedef I8Source<Tile::BM> Rows;
  const uint32_t steps = i8_steps(p.H), parts = (p.F + kCols - 1) / kCols, all = *n_tiles * parts;
  uint32_t j = blockIdx.x / 8, item = item_of(all, parts, j), ahead, now = 0;
  if (item == ~0u) return;
  const uint32_t lane = threadIdx.x & 63, q = lane / 32, col = Tile::w_row() + lane % 32, first = Tile::x_row() + 4 * q;
  const auto same = [](uint32_t r) { return r; };
  const uint64_t experts = (uint64_t)p.E * p.F;
  Rows x(xc, ntok, steps, same);
  I8Source<kCols> g(p.gc, experts, steps, same), u(p.uc, experts, steps, same);
  MoeTile tile = tiles[item / parts], next, after;
  uint32_t f0 = item % parts * kCols, next_f0, id[Rows::kLoads], my_id;
  float sg, su, s;
  // The tile after the next.
  const auto look = [&] {
    j += gridDim.x / 8, ahead = item_of(all, parts, j);
    after = tile_at(tiles, ahead != ~0u ? ahead / parts : 0);
    if (ahead == ~0u) after.count = 0;
  };
  // The next tile's ids; then its rows as the source.
  const auto name = [&] {
#pragma unroll
    for (int i = 0; i < Rows::kLoads; i++) id[i] = order[next.start + (Rows::row(i) < next.count ? Rows::row(i) : 0)];
    my_id = order[next.start + (threadIdx.x < next.count ? threadIdx.x : 0)];
  };
  const auto turn = [&] {
#pragma unroll
    for (int i = 0; i < Rows::kLoads; i++) x.aim(i, Rows::row(i) < next.count ? id[i] / p.K : ntok, steps);
    const uint64_t row = next.count ? (uint64_t)next.expert * p.F + next_f0 : experts;
    g.move(p.gc + row * steps * kI8Row, experts - row, steps);
    u.move(p.uc + row * steps * kI8Row, experts - row, steps);
    s = xs[my_id / p.K];
  };
  next = tile, next_f0 = f0;
  look();
  name();
  turn();
  if (threadIdx.x < Tile::BM) sx[0][threadIdx.x] = s;
  Tile c;
  const auto begin = [&] {
    const bool in = f0 + col < p.F;
    const uint64_t row = (uint64_t)tile.expert * p.F + f0 + col;
    sg = in ? p.gs[row] : 0.0f, su = in ? p.us[row] : 0.0f;
    next = after, next_f0 = ahead % parts * kCols, item = ahead;
    look();
    name();
  };
  const auto done = [&] {
    const __amdgpu_buffer_rsrc_t to =
        mx_buffer((const uint8_t *)(h + (uint64_t)tile.start * pitch), (uint64_t)tile.count * pitch * 4);
    const uint32_t at = f0 + col < p.F ? (first * pitch + f0 + col) * 4 : kNowhere;
    const float limit = kLimit ? p.limit : 0.0f;
#pragma unroll
    for (int m = 0; m < TM; m++)
#pragma unroll
      for (int j = 0; j < 4; j++) {
        const float4 v = *(const float4 *)(sx[now] + first + 32 * m + 8 * j);
        const float r[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int i = 0; i < 4; i++) {
          const float gv = i8_value(c.acc[0][m][4 * j + i], r[i], sg), uv = i8_value(c.acc[1][m][4 * j + i], r[i], su);
          __builtin_amdgcn_raw_buffer_store_b32(__float_as_uint(i8_swiglu(gv, uv, limit)), to, at + (32 * m + 8 * j + i) * pitch * 4, 0,
                                                0);
        }
      }
    now ^= 1;
    if (threadIdx.x < Tile::BM) sx[now][threadIdx.x] = s;
    tile = next, f0 = next_f0;
    return item != ~0u;
  };
  c.template run_items<16 * TM>(
      x0, x1, w0, w1, (steps + 1) / 2 * 2, [&](typename Tile::X &b, uint32_t k) { x.load(k, b.b, steps); },
      [&](typename Tile::W &b, uint32_t k) { g.load(k, b.b, steps), u.load(k, b.b + kCols * kI8Row, steps); }, begin, turn, done);
}

// An item: a tile and 128 of the `cols` rows of down from r0 on. Writes the positions' rows of o, `cols` apart (a multiple of 256).
template <int TM>
__global__ void __launch_bounds__(256) i8_down_tiles(I8Experts p, const int8_t *hc, const float *hs, const MoeTile *tiles,
                                                     const uint32_t *n_tiles, uint32_t r0, uint32_t cols, float *o) {
  typedef I8Tile<TM, 2, 2, true, true> Tile;
  __shared__ typename Tile::X x0;
  __shared__ typename Tile::X x1;
  __shared__ typename Tile::W w0;
  __shared__ typename Tile::W w1;
  __shared__ __align__(16) float sh[2][Tile::BM];
  const uint32_t steps = i8_steps(p.F), parts = cols / Tile::BN, n_items = *n_tiles * parts;
  uint32_t j = blockIdx.x / 8, item = item_of(n_items, parts, j), ahead, now = 0;
  if (item == ~0u) return;
  const uint32_t lane = threadIdx.x & 63, q = lane / 32, col = Tile::w_row() + lane % 32, first = Tile::x_row() + 4 * q;
  const auto same = [](uint32_t r) { return r; };
  const uint64_t all = (uint64_t)p.E * p.H;
  I8Source<Tile::BM> x(hc, 0, steps, same);
  I8Source<Tile::BN> w(p.dc, 0, steps, same);
  MoeTile tile = tiles[item / parts], next, after;
  uint32_t c0 = item % parts * Tile::BN, next_c0;
  float sd[2], s;
  // The tile after the next.
  const auto look = [&] {
    j += gridDim.x / 8, ahead = item_of(n_items, parts, j);
    after = tile_at(tiles, ahead != ~0u ? ahead / parts : 0);
    if (ahead == ~0u) after.count = 0;
  };
  const auto turn = [&] {
    x.move(hc + (uint64_t)next.start * steps * kI8Row, next.count, steps);
    const uint64_t row = next.count ? min((uint64_t)next.expert * p.H + r0 + next_c0, all) : all;
    w.move(p.dc + row * steps * kI8Row, all - row, steps);
    s = hs[next.start + (threadIdx.x < next.count ? threadIdx.x : 0)];
  };
  next = tile, next_c0 = c0;
  look();
  turn();
  if (threadIdx.x < Tile::BM) sh[0][threadIdx.x] = s;
  Tile c;
  const auto begin = [&] {
    const uint64_t row = (uint64_t)tile.expert * p.H + r0 + c0 + col;
#pragma unroll
    for (int f = 0; f < 2; f++) sd[f] = row + f * Tile::kStep < all ? p.ds[row + f * Tile::kStep] : 0.0f;
    next = after, next_c0 = ahead % parts * Tile::BN, item = ahead;
    look();
  };
  const auto done = [&] {
    const __amdgpu_buffer_rsrc_t to = mx_buffer((const uint8_t *)(o + (uint64_t)tile.start * cols), (uint64_t)tile.count * cols * 4);
    const uint32_t at = (first * cols + c0 + col) * 4;
#pragma unroll
    for (int m = 0; m < TM; m++)
#pragma unroll
      for (int j = 0; j < 4; j++) {
        const float4 v = *(const float4 *)(sh[now] + first + 32 * m + 8 * j);
        const float r[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int i = 0; i < 4; i++)
#pragma unroll
          for (int f = 0; f < 2; f++)
            __builtin_amdgcn_raw_buffer_store_b32(__float_as_uint(i8_value(c.acc[f][m][4 * j + i], r[i], sd[f])), to,
                                                  at + (32 * m + 8 * j + i) * cols * 4, f * Tile::kStep * 4, 0);
      }
    now ^= 1;
    if (threadIdx.x < Tile::BM) sh[now][threadIdx.x] = s;
    tile = next, c0 = next_c0;
    return item != ~0u;
  };
  c.template run_items<32 * TM>(
      x0, x1, w0, w1, (steps + 1) / 2 * 2, [&](typename Tile::X &b, uint32_t k) { x.load(k, b.b, steps); },
      [&](typename Tile::W &b, uint32_t k) { w.load(k, b.b, steps); }, begin, turn, done);
}

// ---- few assignments (at most kFew of at most 16 tokens): no sorting, two or three launches. Bound by latency and by reading the
// experts' weights, which go to LDS as whole rows, always some of them on their way: 8 tokens of 10 of 512 experts of 2048 x 512 32
// us (gate and up 17, 3.8 TB/s of the weights; h's quantisation 4; down 14), one token 19.3 (10 and 11), two 21.8, 16 44.5.

constexpr uint32_t kFew = 160;

// The ids (at most kFew; past the experts: E) and the experts they name, each by its first assignment; all 512 threads. The number
// of experts.
struct Named {
  uint32_t first[512];  // an expert's first assignment, then which of those in `used` it is
  uint16_t id[kFew], used[kFew];
  uint32_t counts[8];
};
__device__ __forceinline__ uint32_t name_experts(Named &s, const int32_t *ids, uint32_t A, uint32_t E) {
  const uint32_t lane = threadIdx.x & 63, wave = mx_wave();
  s.first[threadIdx.x] = ~0u;
  uint32_t e = E;
  if (threadIdx.x < A) {
    e = min((uint32_t)ids[threadIdx.x], E);
    s.id[threadIdx.x] = (uint16_t)e;
  }
  __syncthreads();
  if (e < E) atomicMin(s.first + e, threadIdx.x);
  __syncthreads();
  const bool owner = e < E && s.first[e] == threadIdx.x;
  const uint64_t ballot = __ballot(owner);
  if (lane == 0) s.counts[wave] = (uint32_t)__popcll(ballot);
  __syncthreads();
  uint32_t n = 0, at = lanes_below(ballot);
  for (uint32_t v = 0; v < 8; v++) {
    if (v < wave) at += s.counts[v];
    n += s.counts[v];
  }
  if (owner) s.used[at] = (uint16_t)threadIdx.x, s.first[e] = at;
  __syncthreads();
  return n;
}

// The first rank of assignment a's token that names a's expert: its row of h is a's too.
__device__ __forceinline__ uint32_t row_of(const Named &s, uint32_t a, uint32_t K) {
  uint32_t first = a / K * K;
  while (s.id[first] != s.id[a]) first++;
  return first;
}

// This wave's loads but the last kLeft have arrived. (No fence, which would wait for all of them.)
template <int kLeft>
__device__ __forceinline__ void unit_ready() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt(0x0070 | kLeft);  // vmcnt(kLeft) lgkmcnt(0)
  asm volatile("" ::: "memory");
}
// All loads have arrived (LDS is another work-group's after the last wave).
__device__ __forceinline__ void loads_done() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt(0x0f70);
  asm volatile("" ::: "memory");
}

// A unit: 256 bytes of 16 rows, a row's 16-byte pieces exchanged by the row; the operand of four matrix instructions. Each wave has
// three of its own in use or on their way, and needs no barrier for them. Loads past a wave's last unit read nowhere, so that the
// waits count the same everywhere; up to two units that are not there follow the last (with a way out between them the compiler,
// which then no longer tells the buffers' loads apart, waits for all).
constexpr uint32_t kUnit = 256;
constexpr int kUnitLoads = 4;
struct Unit {
  alignas(16) uint8_t c[16 * kUnit];
  __device__ __forceinline__ void read(mx_i4 (&a)[4]) const {
    const uint32_t lane = threadIdx.x & 63, q = lane / 16, r = lane % 16;
#pragma unroll
    for (uint32_t j = 0; j < 4; j++) a[j] = *(const mx_i4 *)(c + r * kUnit + ((4 * j + q) ^ r) * 16);
  }
  // Rows 8 which .. 8 which + 7: those of `from`, `pitch` apart, `bytes` (up to 256) from byte k on.
  __device__ __forceinline__ void load(uint32_t which, __amdgpu_buffer_rsrc_t from, uint32_t pitch, uint32_t k, uint32_t bytes) {
    const uint32_t lane = threadIdx.x & 63;
#pragma unroll
    for (uint32_t j = 0; j < 2; j++) {
      const uint32_t row = which * 8 + 4 * j + lane / 16, at = ((lane % 16) ^ row) * 16;
      lds_dma16(from, at < bytes ? row % 8 * pitch + k + at : kNowhere, c + which * 2048 + j * 1024);
    }
  }
};

// An item: an expert and eight columns of h (eight rows of gate and eight of up: the 16 rows of a matrix instruction, whose 16
// columns are the tokens, whether they use the expert or not). A wave has every so manieth item, or 1 / kSplit of the k axis of one,
// joined in LDS. Each work-group quantises all tokens' x. Writes the rows of h (`pitch` apart, a multiple of 4) of the assignments
// that are their token's first with their expert.
constexpr uint32_t kFewXq = 48 * 1024;  // the tokens' rows of x in LDS

template <uint32_t kX, uint32_t kSplit>
__global__ void __launch_bounds__(512) i8_gate_up_few(I8Experts p, const typename Elem<kX>::T *x, uint64_t stride, uint32_t ntok,
                                                      const int32_t *ids, float *h, uint32_t pitch) {
  __shared__ Unit unit0[8];
  __shared__ Unit unit1[8];
  __shared__ Unit unit2[8];
  __shared__ __align__(16) uint8_t xq[kFewXq + kUnit];  // (a last row's last unit)
  __shared__ int sums[kSplit > 1 ? 8 : 1][16][17];
  __shared__ Named named;
  __shared__ uint32_t most[16], ranks[kFew * 4];  // ranks: [expert][token], a byte: the token's first rank with the expert
  const uint32_t lane = threadIdx.x & 63, wave = mx_wave(), q = lane / 16, r = lane % 16, A = ntok * p.K;
  const uint32_t kpitch = i8_pitch(p.H), lpitch = kpitch + 16, blocks = (p.F + 7) / 8;
  for (uint32_t i = threadIdx.x; i < kFew * 4; i += 512) ranks[i] = ~0u;
  const uint32_t items = name_experts(named, ids, A, p.E) * blocks;
  if (threadIdx.x < A && named.id[threadIdx.x] < p.E && row_of(named, threadIdx.x, p.K) == threadIdx.x)
    ((uint8_t *)ranks)[named.first[named.id[threadIdx.x]] * 16 + threadIdx.x / p.K] = (uint8_t)(threadIdx.x % p.K);
  const uint32_t per = (kpitch + kSplit * kUnit - 1) / (kSplit * kUnit) * kUnit;  // bytes of k a wave
  const uint32_t kfirst = min(wave % kSplit * per, kpitch), kend = min(kfirst + per, kpitch), groups = gridDim.x * 8 / kSplit;
  const auto expert_of = [&](uint32_t item) { return (uint32_t)__builtin_amdgcn_readfirstlane(named.id[named.used[item / blocks]]); };
  uint32_t next = (blockIdx.x * 8 + wave) / kSplit, next_k = kfirst;
  uint32_t item = next, k = kfirst;
  const auto load = [&](Unit &s) {
    const bool real = next < items;
    const uint64_t row = real ? (uint64_t)expert_of(next) * p.F + next % blocks * 8 : 0, rest = ((uint64_t)p.E * p.F - row) * kpitch;
    const uint32_t bytes = real ? min(kend - next_k, kUnit) : 0;
    s.load(0, mx_buffer((const uint8_t *)p.gc + row * kpitch, rest), kpitch, next_k, bytes);
    s.load(1, mx_buffer((const uint8_t *)p.uc + row * kpitch, rest), kpitch, next_k, bytes);
    next_k += kUnit;
    if (next_k >= kend) next_k = kfirst, next += groups;
  };
  float scales[4];  // of the item's four columns that the lane has: gate's in lanes 0 .. 31, up's in the others
  const auto load_scales = [&] {
    if (item >= items) return;
    const float *const from = (q < 2 ? p.gs : p.us) + (uint64_t)expert_of(item) * p.F;
#pragma unroll
    for (uint32_t j = 0; j < 4; j++) scales[j] = from[min(item % blocks * 8 + q % 2 * 4 + j, p.F - 1)];
  };
  load_scales();
  load(unit0[wave]);
  load(unit1[wave]);
  load(unit2[wave]);
  quantize_rows<kX, 4>(ntok, kpitch, p.H, [&](uint32_t i) { return x + i * stride; },
                    [&](uint32_t i, uint32_t c) { return xq + i * lpitch + c; }, most);
  const uint8_t *const xr = xq + min(r, ntok - 1) * lpitch + q * 16;
  // An item's values: lanes 0 .. 31 have gate's sums, lanes 32 on up's, of token r.
  const auto finish = [&](mx_i4 c) {
    const uint32_t f0 = item % blocks * 8 + q % 2 * 4, rank = ((const uint8_t *)ranks)[item / blocks * 16 + r];
    const float sx = i8_scale_of(most[min(r, ntok - 1)]);
    float v[4];
#pragma unroll
    for (uint32_t j = 0; j < 4; j++) {
      const float own = i8_value(c[j], sx, scales[j]);
      v[j] = i8_swiglu(own, __shfl_xor(own, 32, 64), p.limit);  // (of use in the lower half)
    }
    if (q < 2 && r < ntok && rank != 255 && f0 < p.F)
      *(float4 *)(h + (uint64_t)(r * p.K + rank) * pitch + f0) = make_float4(v[0], v[1], v[2], v[3]);
  };
  mx_i4 acc = {0, 0, 0, 0};
  const auto use = [&](Unit &s) {
    unit_ready<2 * kUnitLoads>();
    mx_i4 a[4], b[4];
    s.read(a);
#pragma unroll
    for (uint32_t j = 0; j < 4; j++) b[j] = *(const mx_i4 *)(xr + k + j * 64);  // (past a row's end: times zeros)
#pragma unroll
    for (uint32_t j = 0; j < 4; j++) acc = i8_mfma16(a[j], b[j], acc);
    load(s);
    k += kUnit;
    if (k < kend) return;
    if (kSplit == 1) {
      if (item < items) finish(acc);
      acc = mx_i4{0, 0, 0, 0};
    }
    k = kfirst, item += groups;
    if (kSplit == 1) load_scales();
  };
  if (kSplit == 1) {
#pragma unroll 1
    while (item < items) {
      use(unit0[wave]);
      use(unit1[wave]);
      use(unit2[wave]);
    }
    loads_done();
  } else {  // (one item a wave at most)
    const uint32_t mine = item;
    if (kfirst < kend) {
#pragma unroll 1
      while (item == mine && item < items) {
        use(unit0[wave]);
        use(unit1[wave]);
        use(unit2[wave]);
      }
    }
    loads_done();
#pragma unroll
    for (uint32_t j = 0; j < 4; j++) sums[wave][4 * q + j][r] = acc[j];
    __syncthreads();
    if (wave % kSplit != 0 || mine >= items) return;
#pragma unroll
    for (uint32_t s = 1; s < kSplit; s++)
#pragma unroll
      for (uint32_t j = 0; j < 4; j++) acc[j] += sums[wave + s][4 * q + j][r];
    item = mine;
    finish(acc);
  }
}

// A work-group takes every gridDim-th eight rows of down, y's eight columns, for all assignments. A wave has every eighth pair of the
// experts that are named, whose eight rows each are the 16 rows of a matrix instruction; its columns are eight assignments of the
// one and eight of the other, of which half of the products count. kOwn: it quantises the rows of h itself, at most kFewOwn values
// (a launch for that is 3 us; more values take each work-group as long: 8 tokens of 10 ranks 38 us so, 32 with the launch). kUnits:
// the units of a wave in LDS, three if h's rows leave them room.
constexpr uint32_t few_hq(int units) { return (units == 3 ? 48 : 80) * 1024; }  // the assignments' rows of h in LDS
constexpr uint32_t kFewOwn = 512 * 4 * 8;
constexpr uint32_t kTerms = (kFew * 8 + 511) / 512;

template <uint32_t kType, bool kOwn, int kUnits>
__global__ void __launch_bounds__(512) i8_down_few(I8Experts p, const float *h, uint32_t hpitch, const int8_t *hc, const float *hs,
                                                   const int32_t *ids, const float *w, uint32_t ntok, typename Elem<kType>::T *y,
                                                   uint64_t stride) {
  __shared__ Unit unit0[8];
  __shared__ Unit unit1[8];
  __shared__ Unit unit2[kUnits == 3 ? 8 : 1];
  __shared__ __align__(16) uint8_t hq[few_hq(kUnits) + 1024];  // a row's 16-byte pieces exchanged by the row
  __shared__ __align__(16) int o[kFew * 8];
  __shared__ Named named;
  __shared__ uint16_t member[8][2][kFew], row[kFew];
  __shared__ float weight[kFew];
  __shared__ uint32_t most[kFew];
  const uint32_t lane = threadIdx.x & 63, wave = mx_wave(), q = lane / 16, r = lane % 16, A = ntok * p.K;
  const uint32_t pitch = i8_pitch(p.F), blocks = (p.H + 7) / 8;
  const uint32_t n = name_experts(named, ids, A, p.E), pairs = (n + 1) / 2;
  // The two experts of a pair (the second one may be none: n is odd).
  const auto expert_of = [&](uint32_t pair, uint32_t which) {
    const uint32_t i = pair * 2 + which;
    return i < n ? (uint32_t)__builtin_amdgcn_readfirstlane(named.id[named.used[i]]) : p.E;
  };
  uint32_t next_pair = 0, next_k = 0, r0 = 0;
  const auto load = [&](Unit &s) {
#pragma unroll
    for (uint32_t which = 0; which < 2; which++) {
      const uint32_t e = expert_of(next_pair, which);
      const uint64_t first = (uint64_t)min(e, p.E - 1) * p.H + r0, rest = (uint64_t)p.E * p.H - first;
      s.load(which, mx_buffer((const uint8_t *)p.dc + first * pitch, rest * pitch), pitch, next_k,
             e < p.E ? min(pitch - next_k, kUnit) : 0);
    }
    next_k += kUnit;
    if (next_k >= pitch) next_k = 0, next_pair += 8;
  };
  uint32_t pair = 0, k = 0, nm[2] = {0, 0};
  const auto use = [&](Unit &s) {
    unit_ready<(kUnits - 1) * kUnitLoads>();
    if (k == 0) {  // the experts' assignments
#pragma unroll
      for (uint32_t which = 0; which < 2; which++) {
        const uint32_t ex = expert_of(pair, which);
        nm[which] = 0;
#pragma unroll 1
        for (uint32_t a0 = 0; a0 < A; a0 += 64) {
          const bool is = a0 + lane < A && named.id[min(a0 + lane, A - 1)] == ex && ex < p.E;
          const uint64_t bal = __ballot(is);
          if (is) member[wave][which][nm[which] + lanes_below(bal)] = (uint16_t)(a0 + lane);
          nm[which] += (uint32_t)__popcll(bal);
        }
      }
      __builtin_amdgcn_s_waitcnt(0xc07f);
      __builtin_amdgcn_wave_barrier();
    }
    mx_i4 a[4];
    s.read(a);
    const uint32_t mine = r / 8, many = mine ? nm[1] : nm[0];
#pragma unroll 1
    for (uint32_t m0 = 0; m0 < max(nm[0], nm[1]); m0 += 8) {
      const bool there = m0 + r % 8 < many;
      const uint32_t as = there ? member[wave][mine][m0 + r % 8] : 0;
      const bool counts = there && q / 2 == mine;  // (the other rows are the other expert's)
      const uint32_t hr = row[as];
      const uint8_t *const from = hq + hr * pitch + k;
      mx_i4 c = {0, 0, 0, 0};
      int4 *to = (int4 *)(o + as * 8 + q % 2 * 4);
      if (k != 0 && counts) {
        const int4 v = *to;
        c = mx_i4{v.x, v.y, v.z, v.w};
      }
#pragma unroll
      for (uint32_t j = 0; j < 4; j++)  // (past a row's end: times zeros)
        c = i8_mfma16(a[j], *(const mx_i4 *)(from + ((4 * j + q) ^ (hr % 8)) * 16), c);
      if (counts) *to = make_int4(c[0], c[1], c[2], c[3]);
    }
    load(s);
    k += kUnit;
    if (k >= pitch) k = 0, pair += 8;
  };
  for (uint32_t b = blockIdx.x; b < blocks; b += gridDim.x) {
    r0 = b * 8, next_pair = pair = wave, next_k = k = 0;
    // (Rows of assignments without an expert, or not their token's first with it, hold what nobody reads.)
    if (!kOwn && b == blockIdx.x)
      for (uint32_t i = wave * 1024; i < A * pitch; i += 8 * 1024) {
        const uint32_t at = i + lane * 16, hr = at / pitch, piece = (at - hr * pitch) / 16;
        lds_dma16(mx_buffer((const uint8_t *)hc, A * pitch), hr * pitch + (piece ^ (hr % 8)) * 16, hq + i);
      }
    load(unit0[wave]);
    load(unit1[wave]);
    if constexpr (kUnits == 3) load(unit2[wave]);
    if (b == blockIdx.x) {
      if (threadIdx.x < A) {
        const bool on = named.id[threadIdx.x] < p.E;
        row[threadIdx.x] = (uint16_t)row_of(named, threadIdx.x, p.K), weight[threadIdx.x] = on ? w[threadIdx.x] : 0.0f;
      }
      if (kOwn) {
        quantize_rows<QT_F32, 4>(A, pitch, p.F, [&](uint32_t i) { return h + (uint64_t)i * hpitch; },
                              [&](uint32_t i, uint32_t c) { return hq + i * pitch + ((c / 16) ^ (i % 8)) * 16 + c % 16; }, most);
      } else {
        asm volatile("" ::: "memory");
        __builtin_amdgcn_s_waitcnt(0x0070 | kUnits * kUnitLoads);  // (all but the units: the rows of h)
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
      }
    }
    // The scales of the sums that the thread turns into values.
    float hscale[kTerms], dscale[kTerms];
#pragma unroll
    for (uint32_t j = 0; j < kTerms; j++) {
      const uint32_t i = min(threadIdx.x + j * 512, A * 8 - 1), a = i / 8, ex = min((uint32_t)named.id[a], p.E - 1);
      hscale[j] = kOwn ? i8_scale_of(most[row[a]]) : hs[row[a]];
      dscale[j] = p.ds[min((uint64_t)ex * p.H + r0 + i % 8, (uint64_t)p.E * p.H - 1)];
    }
    asm volatile("" ::: "memory");
#pragma unroll 1
    while (pair < pairs) {
      use(unit0[wave]);
      use(unit1[wave]);
      if constexpr (kUnits == 3) use(unit2[wave]);
    }
    loads_done();
    __syncthreads();
#pragma unroll
    for (uint32_t j = 0; j < kTerms; j++) {
      const uint32_t i = threadIdx.x + j * 512;
      if (i < A * 8) o[i] = named.id[i / 8] < p.E ? __float_as_int(i8_value(o[i], hscale[j], dscale[j])) : 0;
    }
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < ntok * 8; i += 512) {
      const uint32_t t = i / 8, c = i % 8;
      float s = 0.0f;
#pragma unroll 8
      for (uint32_t a = t * p.K; a < (t + 1) * p.K; a++) s = __builtin_fmaf(weight[a], __int_as_float(o[a * 8 + c]), s);
      if (r0 + c < p.H) y[(uint64_t)t * stride + r0 + c] = (typename Elem<kType>::T)s;
    }
    __syncthreads();  // (o)
  }
}

}  // namespace c0ven

using namespace c0ven;

namespace {

void check_experts(const moe_i8_experts *e, uint32_t ntok) {
  op_require(e != nullptr, "null argument");
  op_require(e->n_embd >= 1 && e->n_embd <= 16384 && e->n_ff >= 1 && e->n_ff <= 16384, "n_embd and n_ff must be 1..16384");
  op_require(e->n_expert >= 1 && e->n_expert <= 512, "n_expert must be 1..512");
  op_require(e->n_used >= 1 && e->n_used <= 16, "n_used must be 1..16");
  op_require(e->swiglu_limit >= 0.0f && e->swiglu_limit < INFINITY, "swiglu_limit must be finite and not negative");
  op_require(ntok <= 16384, "at most 16384 tokens");
  for (const moe_i8_matrix *m : {&e->gate, &e->up, &e->down}) op_i8(m);
  op_require(e->gate.rows == e->n_ff && e->gate.cols == e->n_embd && e->up.rows == e->n_ff && e->up.cols == e->n_embd &&
                 e->down.rows == e->n_embd && e->down.cols == e->n_ff,
             "gate and up must be n_ff x n_embd, down n_embd x n_ff");
  op_require(op_float(e->x_type) && op_float(e->y_type), "the element type must be QT_F32, QT_F16 or QT_BF16");
}

// How a call runs. Few assignments, whose rows of h fit LDS, without sorting them: 16 tokens of 10 of 512 experts of 2048 x 512 44
// us, sorted 49; of 16 experts 28 and 35; but 12 of 512 of 2560 x 640 64 and 63.
constexpr uint64_t kTurnBytes = 256 << 20;
constexpr uint32_t kCus = 256;  // work-groups that fill the device where LDS holds one a CU

struct Plan {
  uint32_t A, rows, hpitch, pitch, chunk, max_tiles;
  bool few;
  uint64_t xc, xs, h, hc, hs, o, sort, order, places, offsets, tiles, n_tiles, bytes;  // the work buffer's parts

  Plan(const moe_i8_experts &e, uint32_t T) {
    A = T * e.n_used;
    few = !A || (T <= 16 && A <= kFew && e.n_embd >= 8 && T * (i8_pitch(e.n_embd) + 16) <= kFewXq && A * i8_pitch(e.n_ff) <= few_hq(2));
    // Tiles of 64 or 128 positions: the more an expert has on average, the fewer times its weights are read, as long as the tiles
    // are enough for the CUs. 2048 tokens of 10 of 512 experts (40 each) 399 and 410 us, 1024 of 8 of 128 (64) 136 and 141; 4096 (80)
    // 545 and 501, with skewed experts 411 and 388; 1000 tokens of 4 of 8 (500, 250 pieces) 50 and 52, 2000 (500 pieces) 81 and 79,
    // 4096 159 and 149. (Of 32, 30 of 10 of 512 take 53.6 and with 64 53.7, 300 both 310, 301 of a skewed router 153 and 138. Of
    // 256, with i8_gemm's five buffers, 4096 of 4 of 8 were 178 and with 128 163: h and the values go out after 4 or 16 stages.)
    rows = A / e.n_expert < 72 || (uint64_t)A / 128 * ((e.n_ff + 63) / 64) < 400 ? 64 : 128;
    hpitch = (e.n_ff + 3) / 4 * 4;
    pitch = (e.n_embd + 255) / 256 * 256;
    // The values of all assignments at once, or in turns of about 256 MB each, the last-level cache's size (4096 tokens of 10 of 512
    // experts in two turns 378 us, on another card 403; before the tiles' last steps all at once 438, in turns of 256 MB 437, of 128 450, of 64 495).
    const uint64_t turns = (4ull * A * pitch + kTurnBytes - 1) / kTurnBytes;
    chunk = few ? pitch : (uint32_t)((pitch / 256 + turns - 1) / turns * 256);
    max_tiles = std::min(A, e.n_expert + A / rows);
    uint64_t at = 0;
    const auto part = [&](uint64_t n) {
      const uint64_t was = at;
      at += (n + 255) / 256 * 256;
      return was;
    };
    h = part((uint64_t)A * hpitch * 4), hc = part(i8_bytes(A, e.n_ff)), hs = part((uint64_t)A * 4);
    if (!few) {
      xc = part(i8_bytes(T, e.n_embd)), xs = part((uint64_t)T * 4);
      o = part((uint64_t)A * chunk * 4);
      sort = part(sort_bytes(A, e.n_expert)), order = part((uint64_t)A * 4), places = part((uint64_t)A * 4);
      offsets = part((e.n_expert + 1) * 4ull);
      tiles = part((uint64_t)max_tiles * sizeof(MoeTile)), n_tiles = part(4);
    }
    bytes = at;
  }
};

}  // namespace

extern "C" {

MOE_API uint64_t moe_i8_experts_work_bytes(const moe_i8_experts *e, uint32_t ntok) {
  uint64_t n = 0;
  (void)op_guarded([&] {
    check_experts(e, ntok);
    n = Plan(*e, ntok).bytes;
  });
  return n;
}

MOE_API moe_status moe_i8_experts_async(const moe_i8_experts *e, const void *x, uint64_t x_stride, uint32_t ntok,
                                        const int32_t *ids, const float *w, void *y, uint64_t y_stride, void *work,
                                        uint64_t work_bytes, void *stream) {
  return op_guarded([&] {
    check_experts(e, ntok);
    const uint32_t H = e->n_embd, F = e->n_ff, E = e->n_expert, K = e->n_used, A = ntok * K;
    op_rows(x, x_stride, ntok, H, e->x_type);
    op_rows(y, y_stride, ntok, H, e->y_type);
    op_require(((ids && w) || !ntok) && op_aligned(ids, 4) && op_aligned(w, 4), "null or misaligned ids or w");
    const Plan at(*e, ntok);
    op_work(work, work_bytes, at.bytes);
    if (!ntok) return;
    OnDevice on(e->device);
    uint8_t *b = (uint8_t *)work;
    const I8Experts p{e->gate.codes, e->up.codes, e->down.codes, e->gate.scales, e->up.scales, e->down.scales, E, K, H, F,
                      e->swiglu_limit};
    float *h = (float *)(b + at.h);
    const moe_i8_matrix hq{(int8_t *)(b + at.hc), (float *)(b + at.hs), A, F};
    if (at.few) {
      // The k axis is split where the items leave half of the waves or more without one.
      const uint32_t items = std::min(A, E) * ((F + 7) / 8), waves = kCus * 8;
      op_by_type(e->x_type, [&](auto t) {
        constexpr uint32_t kX = decltype(t)::value;
        const auto run = [&](auto kernel, uint32_t split) {
          op_launch(kernel, std::min((items * split + 7) / 8, kCus), 512, stream, p, (const typename Elem<kX>::T *)x, x_stride, ntok,
                    ids, h, at.hpitch);
        };
        if (items * 4 <= waves)
          run(i8_gate_up_few<kX, 4>, 4);
        else if (items * 2 <= waves)
          run(i8_gate_up_few<kX, 2>, 2);
        else
          run(i8_gate_up_few<kX, 1>, 1);
      });
      const bool own = F >= 8 && A * i8_pitch(F) <= kFewOwn;
      if (!own) i8_quantize_launch(QT_F32, h, at.hpitch, hq, nullptr, stream);
      op_by_type(e->y_type, [&](auto t) {
        constexpr uint32_t kY = decltype(t)::value;
        const auto run = [&](auto kernel) {
          op_launch(kernel, std::min((H + 7) / 8, kCus), 512, stream, p, (const float *)h, at.hpitch, (const int8_t *)hq.codes,
                    (const float *)hq.scales, ids, w, ntok, (typename Elem<kY>::T *)y, y_stride);
        };
        if (own)
          run(i8_down_few<kY, true, 3>);
        else if (A * i8_pitch(F) <= few_hq(3))
          run(i8_down_few<kY, false, 3>);
        else
          run(i8_down_few<kY, false, 2>);
      });
      return;
    }
    int32_t *order = (int32_t *)(b + at.order), *places = (int32_t *)(b + at.places);
    uint32_t *offsets = (uint32_t *)(b + at.offsets), *nt = (uint32_t *)(b + at.n_tiles);
    MoeTile *tiles = (MoeTile *)(b + at.tiles);
    float *o = (float *)(b + at.o);
    const moe_i8_matrix xq{(int8_t *)(b + at.xc), (float *)(b + at.xs), ntok, H};
    const SortOut sorted{order, places, offsets, tiles, nt, at.rows};
    const uint32_t slices = slices_of(A);  // (of kSlice ids: A is at most 2^18)
    op_by_type(e->x_type, [&](auto t) {
      constexpr uint32_t kX = decltype(t)::value;
      const bool wide = H > 2048;
      const auto run = [&](auto kernel) {
        op_launch(kernel, slices + (wide ? ntok : (ntok + 15) / 16), 1024, stream, ids, A, E, slices, (uint32_t *)(b + at.sort), sorted,
                  (const typename Elem<kX>::T *)x, x_stride, ntok, H, xq.codes, xq.scales);
      };
      if (slices == 1)
        wide ? run(i8_prepare<kX, true, false>) : run(i8_prepare<kX, false, false>);
      else
        wide ? run(i8_prepare<kX, true, true>) : run(i8_prepare<kX, false, true>);
    });
    if (slices > 1) sort_place_launch(ids, A, E, sorted, b + at.sort, stream);
    const auto run = [&](auto gate_up, auto down, uint32_t at_once) {
      const uint64_t bn = 128, parts = (F + bn / 2 - 1) / (bn / 2);
      const auto blocks = [&](uint64_t n) { return std::min<uint64_t>(item_blocks(at.max_tiles * n, n), at_once); };
      op_launch(gate_up, blocks(parts), 256, stream, p, (const int8_t *)xq.codes, (const float *)xq.scales, ntok, (const int32_t *)order,
                (const MoeTile *)tiles, (const uint32_t *)nt, h, at.hpitch);
      i8_quantize_launch(QT_F32, h, at.hpitch, hq, offsets + E, stream);
      for (uint32_t c = 0; c < at.pitch; c += at.chunk) {
        const uint32_t n = std::min(at.chunk, at.pitch - c);
        op_launch(down, blocks(n / bn), 256, stream, p, (const int8_t *)hq.codes, (const float *)hq.scales, (const MoeTile *)tiles,
                  (const uint32_t *)nt, c, n, o);
        combine_launch(QT_F32, o, n, ntok, K, std::min(n, H - c), places, w, e->y_type, (uint8_t *)y + (uint64_t)c * op_size(e->y_type),
                       y_stride, stream);
      }
    };
    const auto tiles_of = [&](auto limit) {
      constexpr bool kLimit = decltype(limit)::value;
      if (at.rows == 64) run(i8_gate_up_tiles<1, kLimit>, i8_down_tiles<1>, 3 * kCus);
      if (at.rows == 128) run(i8_gate_up_tiles<2, kLimit>, i8_down_tiles<2>, 2 * kCus);
    };
    e->swiglu_limit > 0.0f ? tiles_of(std::true_type()) : tiles_of(std::false_type());
  });
}

}  // extern "C"
