// The experts of routed tokens in MX4 (moe_mx4_experts_async).
//
// Many tokens, in four launches (mx4_prepare, gate/up, down, combine; down and combine again for each part of the columns):
// the assignments (token * n_used + rank) are sorted by expert and cut into MoeTiles; gate and up of a tile are one product
// whose epilogue applies the SwiGLU and quantises h, 32 neighbours of a row being in one wave's registers; down follows on the
// positions' rows, its fp32 sums go to the assignments' rows, and a last kernel adds each token's in rank order. 301 tokens of
// 10 of 512 skewed experts, 2560 x 640, fp16: gate/up 50 us, down 34, combine 7, prepare 5; bound by the experts' weights (274
// MB, 53 us at 5.2 TB/s). 4096 tokens, 2048 x 512: gate/up 126 us (a stage's latency at three work-groups a CU; its
// instructions and LDS are at a third), down 87 + 33 and combine 45 + 14 in two parts (335 MB of sums written and read back at 5.6 TB/s),
// prepare 15.
#include "../../include/c0ven_moe_tile.h"
#include "mx4.h"
#include "mx4_api.h"
#include "mx4_gemm.h"
#include "ops.h"

#include <algorithm>

namespace c0ven {

// silu(g) u with the limit of moe_config.swiglu_limit; NaNs stay.
__device__ __forceinline__ float mx_swiglu(float g, float u, float limit) {
  if (limit > 0.0f) {
    g = g > limit ? limit : g;
    u = u > limit ? limit : u < -limit ? -limit : u;
  }
  return g / (1.0f + exp_f32(-g)) * u;
}

// ---- the assignments by expert, and x in MX4

constexpr uint32_t kSlice = 4096;   // ids a work-group sorts
constexpr uint32_t kGroups = 4096;  // groups of eight values a work-group quantises

// The first `slices` work-groups: each takes every id (counting all of them costs a work-group less than a launch for the
// counts does), then puts its slice's assignments to their places (order[place] = assignment; within an expert by slice);
// the first one writes the tiles of at most `rows` places each. The others quantise x, of mx_steps(H) steps.
template <uint32_t kX>
__global__ void __launch_bounds__(1024) mx4_prepare(const int32_t *ids, uint32_t A, uint32_t E, uint32_t slices, uint32_t rows,
                                                    uint32_t *order, MoeTile *tiles, uint32_t *n_tiles,
                                                    const typename Elem<kX>::T *x, uint64_t stride, uint32_t ntok, uint32_t H,
                                                    uint8_t *xc, uint8_t *xs) {
  const uint32_t e = threadIdx.x;
  if (blockIdx.x >= slices) {
    const uint32_t per = mx_steps(H) * 16, end = ntok * per, g0 = (blockIdx.x - slices) * kGroups + e;
    float v[kGroups / 1024][8];
#pragma unroll
    for (uint32_t i = 0; i < kGroups / 1024; i++) {
      const uint32_t g = min(g0 + i * 1024, end - 1);
      load8<kX>(x + g / per * stride, g % per * 8, H, v[i]);
    }
#pragma unroll
    for (uint32_t i = 0; i < kGroups / 1024; i++) {
      const uint32_t g = g0 + i * 1024;
      uint32_t s;
      const uint32_t c = mx_quantize8(v[i], s);
      if (g >= end) break;
      ((uint32_t *)xc)[g] = c;
      if (g % 4 == 0) xs[g / 4] = (uint8_t)s;
    }
    return;
  }
  __shared__ uint32_t before[512], other[512];  // an expert's assignments: in the slices before this one, elsewhere
  __shared__ uint32_t sums[2][8];
  const uint32_t first = blockIdx.x * kSlice, end = min(A, first + kSlice);
  if (e < 512) before[e] = other[e] = 0;
  __syncthreads();
  for (uint32_t i0 = e; i0 < A; i0 += 8 * 1024) {
    uint32_t id[8];
#pragma unroll
    for (uint32_t j = 0; j < 8; j++) id[j] = i0 + j * 1024 < A ? (uint32_t)ids[i0 + j * 1024] : ~0u;
#pragma unroll
    for (uint32_t j = 0; j < 8; j++)
      if (id[j] < E) atomicAdd((i0 + j * 1024 < first ? before : other) + id[j], 1u);
  }
  __syncthreads();
  const uint32_t was = e < 512 ? before[e] : 0, all = e < 512 ? was + other[e] : 0, n = (all + rows - 1) / rows;
  uint32_t place = all, tile = n;  // their sums up to this expert
  for (uint32_t d = 1; d < 64; d *= 2) {
    const uint32_t p = (uint32_t)__shfl_up((int)place, d, 64), t = (uint32_t)__shfl_up((int)tile, d, 64);
    if (e % 64 >= d) place += p, tile += t;
  }
  if (e < 512 && e % 64 == 63) sums[0][e / 64] = place, sums[1][e / 64] = tile;
  __syncthreads();
  if (e < 512) {
    for (uint32_t v = 0; v < e / 64; v++) place += sums[0][v], tile += sums[1][v];
    before[e] = place - all + was;
    if (blockIdx.x == 0) {
      for (uint32_t j = 0; j < n; j++)
        tiles[tile - n + j] = MoeTile{e, e, place - all + j * rows, min(rows, all - j * rows)};
      if (e == 511) *n_tiles = tile;
    }
  }
  __syncthreads();
  for (uint32_t i = first + e; i < end; i += 1024) {
    const uint32_t id = (uint32_t)ids[i];
    if (id < E) order[atomicAdd(before + id, 1u)] = i;
  }
}

// ---- the products

struct MxExperts {
  const uint8_t *gc, *gs, *uc, *us, *dc, *ds;
  uint32_t E, K, H, F;
  float limit;
};

// A launch's work-groups to its items (parts a tile) so that an XCD (work-groups go to the eight in turn) has runs of four
// tiles: an expert's tiles share its weights in that L2, while the experts with one tile are dealt over all of them (4096
// tokens of 10 of 512 experts 392 us, with the items in order 430; of 4 of 16 experts 114 and 119). ~0: none.
constexpr uint32_t kTileRun = 4;
__device__ __forceinline__ uint32_t item_of(uint32_t all, uint32_t parts) {
  const uint32_t run = kTileRun * parts, j = blockIdx.x / 8, id = (j / run * 8 + blockIdx.x % 8) * run + j % run;
  return id < all ? id : ~0u;
}
// The work-groups that cover `all` items.
inline uint64_t item_blocks(uint64_t all, uint64_t parts) {
  const uint64_t run = kTileRun * parts;
  return (all + 8 * run - 1) / (8 * run) * (8 * run);
}

// An item: a tile and 32 WN columns of h (their rows of gate and of up). Writes the places' rows of h in MX4.
template <int TM, int WM>
__global__ void __launch_bounds__(256) mx4_gate_up_tiles(MxExperts p, const uint8_t *xc, const uint8_t *xs, uint32_t ntok,
                                                         const uint32_t *order, const MoeTile *tiles, const uint32_t *n_tiles,
                                                         uint8_t *hc, uint8_t *hs) {
  typedef MxTile<TM, 2, WM, true> Tile;
  constexpr uint32_t kCols = Tile::BN / 2;
  __shared__ typename Tile::Stage s0;
  __shared__ typename Tile::Stage s1;
  __shared__ typename Tile::Scales scales;
  const uint32_t steps = mx_steps(p.H), hsteps = mx_steps(p.F), parts = hsteps * 128 / kCols, item = item_of(*n_tiles * parts, parts);
  if (item == ~0u) return;
  const MoeTile tile = tiles[item / parts];
  const uint32_t f0 = item % parts * kCols, stages = (steps + 1) / 2;
  const uint64_t row = (uint64_t)tile.expert * p.F + f0, rest = (uint64_t)p.E * p.F - min(row, (uint64_t)p.E * p.F);
  const auto same = [](uint32_t r) { return r; };
  const MxSource<Tile::BM> x(xc, xs, ntok, steps, [&](uint32_t r) { return order[tile.start + min(r, tile.count - 1)] / p.K; });
  const MxSource<kCols> g(p.gc + row * steps * 64, p.gs + row * steps * 4, rest, steps, same);
  const MxSource<kCols> u(p.uc + row * steps * 64, p.us + row * steps * 4, rest, steps, same);
  Tile c;
  c.run(
      s0, s1, scales, stages,
      [&](typename Tile::Stage &s, uint32_t k) { g.load(k, s.w), u.load(k, s.w + kCols * 128), x.load(k, s.x); },
      [&](typename Tile::Scales &s, uint32_t k) {
        g.load_scales(k, s.w), u.load_scales(k, s.w + kCols * 4), x.load_scales(k, s.x);
      });
  // Lane l has 16 of its token's 32 columns of a wave (8 j + 4 (l / 32) + i), lane l ^ 32 the others.
  const uint32_t lane = threadIdx.x & 63, q = lane / 32, col = f0 + Tile::w_row();
#pragma unroll
  for (int m = 0; m < TM; m++) {
    float h[16];
    uint32_t most = 0;
#pragma unroll
    for (int i = 0; i < 16; i++) {
      h[i] = mx_swiglu(c.acc[0][m][i], c.acc[1][m][i], p.limit);
      if (col + 8 * (i / 4) + 4 * q + i % 4 >= p.F) h[i] = 0.0f;
      most = max(most, __float_as_uint(h[i]) & 0x7fffffffu);
    }
    most = max(most, (uint32_t)__shfl_xor((int)most, 32, 64));
    const uint32_t s = mx_scale_of(most);
    const uint32_t a = s == 255 ? 0u : mx_codes8(h, s), b = s == 255 ? 0u : mx_codes8(h + 8, s);
    const uint32_t oa = (uint32_t)__shfl_xor((int)a, 32, 64), ob = (uint32_t)__shfl_xor((int)b, 32, 64);
    const uint32_t r = Tile::x_row() + 32 * m + lane % 32;
    if (q == 0 && r < tile.count) {
      const uint64_t at = (uint64_t)(tile.start + r) * hsteps * 4 + col / 32;
      *(uint4 *)(hc + at * 16) = make_uint4((a & 0xffff) | oa << 16, (a >> 16) | (oa & 0xffff0000u), (b & 0xffff) | ob << 16,
                                            (b >> 16) | (ob & 0xffff0000u));
      hs[at] = (uint8_t)s;
    }
  }
}

// An item: a tile and BN of the `cols` rows of down from r0 on. Writes the sums to the assignments' rows of o, `cols` apart (a
// multiple of 256): a lane has a column of 16 rows, so that a store is of whole lines (two rows of 32 columns; with a row's
// four neighbours a lane it was 32 rows of 32 bytes: 4096 tokens 172 us in all, now 128).
template <int TM, int WM>
__global__ void __launch_bounds__(256) mx4_down_tiles(MxExperts p, const uint8_t *hc, const uint8_t *hs, uint32_t A,
                                                      const uint32_t *order, const MoeTile *tiles, const uint32_t *n_tiles,
                                                      uint32_t r0, uint32_t cols, float *o) {
  typedef MxTile<TM, 2, WM, true, true> Tile;
  __shared__ typename Tile::Stage s0;
  __shared__ typename Tile::Stage s1;
  __shared__ typename Tile::Scales scales;
  __shared__ __align__(16) uint32_t place[Tile::BM];  // where a row of the tile goes, in bytes (kNowhere: dropped)
  const uint32_t steps = mx_steps(p.F), parts = cols / Tile::BN, item = item_of(*n_tiles * parts, parts);
  if (item == ~0u) return;
  const MoeTile tile = tiles[item / parts];
  const uint32_t c0 = item % parts * Tile::BN;
  const uint64_t row = (uint64_t)tile.expert * p.H + r0 + c0, rest = (uint64_t)p.E * p.H - min(row, (uint64_t)p.E * p.H);
  const auto same = [](uint32_t r) { return r; };
  const MxSource<Tile::BM> x(hc, hs, A, steps, [&](uint32_t r) { return tile.start + min(r, tile.count - 1); });
  const MxSource<Tile::BN> w(p.dc + row * steps * 64, p.ds + row * steps * 4, rest, steps, same);
  const uint32_t lane = threadIdx.x & 63, q = lane / 32;
  if (threadIdx.x < Tile::BM)
    place[threadIdx.x] = threadIdx.x < tile.count ? order[tile.start + threadIdx.x] * cols * 4 : kNowhere;
  Tile c;
  c.run(
      s0, s1, scales, (steps + 1) / 2,
      [&](typename Tile::Stage &s, uint32_t k) { w.load(k, s.w), x.load(k, s.x); },
      [&](typename Tile::Scales &s, uint32_t k) { w.load_scales(k, s.w), x.load_scales(k, s.x); });
  const __amdgpu_buffer_rsrc_t to = mx_buffer((const uint8_t *)o, (uint64_t)A * cols * 4);
  const uint32_t col = (c0 + Tile::w_row() + lane % 32) * 4;
#pragma unroll
  for (int m = 0; m < TM; m++)
#pragma unroll
    for (int j = 0; j < 4; j++) {
      const uint4 v = *(const uint4 *)(place + Tile::x_row() + 32 * m + 8 * j + 4 * q);
      const uint32_t at[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
      for (int i = 0; i < 4; i++)
#pragma unroll
        for (int f = 0; f < 2; f++)
          __builtin_amdgcn_raw_buffer_store_b32(__float_as_uint(c.acc[f][m][4 * j + i]), to, at[i] + col, f * Tile::kStep * 4, 0);
    }
}

// ---- few assignments (at most kFew): no sorting, two launches. Bound by latency and by reading the experts' weights, which
// go to LDS as whole rows (a matrix instruction's operand straight from memory is 16 rows of 64 bytes, a clock a lane; whole
// rows are 4 lanes a clock): all that a work-group needs is on its way at once.

constexpr uint32_t kFew = 160;

// What lane l of 64 holds (flag) as the number of lanes below it that do.
__device__ __forceinline__ uint32_t lanes_below(uint64_t ballot) {
  return __builtin_amdgcn_mbcnt_hi((uint32_t)(ballot >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)ballot, 0u));
}

// A work-group: an expert and 32 columns of h, for the tokens that use the expert, eight at a time: the assignment that is
// the first with its expert does the work, the others' work-groups leave. Quantises x itself (while the weights come) and
// writes the assignments' rows of h in MX4. Four waves share the k axis, kSteps steps of 128 at a time (all of n_embd, where
// it is not longer); the sums are joined in LDS. kSteps 16 where that is all of n_embd: two work-groups a CU, with the LDS of
// 24 one (8 tokens of 10 of 512 experts 41 us, 49; one token 14, 14). One token: 6.5 us of the call's 12.7; 8 tokens with skewed
// experts 11.7 of 22.5.
template <uint32_t kX, int kSteps>
__global__ void __launch_bounds__(256) mx4_gate_up_few(MxExperts p, const typename Elem<kX>::T *x, uint64_t stride,
                                                       const int32_t *ids, uint32_t A, uint8_t *hc, uint8_t *hs) {
  constexpr uint32_t kTok = 8, kPitch = kSteps * 64, kXPitch = kSteps * 64 + 16;
  __shared__ __align__(16) uint8_t wc[64 * kPitch];     // gate's 32 rows, up's; a row's 16-byte pieces exchanged by r % 16
  __shared__ __align__(16) uint32_t wsc[64 * kSteps];   // their scales, a word a step
  constexpr uint32_t kXBytes = kTok * kXPitch + kTok * kSteps * 4, kSumBytes = 4 * 64 * kTok * 4;
  __shared__ __align__(16) uint8_t shared[kXBytes > kSumBytes ? kXBytes : kSumBytes];  // x's rows, then the waves' sums
  __shared__ float h[kTok][33];
  __shared__ uint16_t member[kFew];
  __shared__ uint32_t counts[4];
  uint8_t *xc = shared;
  uint32_t *xsc = (uint32_t *)(shared + kTok * kXPitch);
  float *sums = (float *)shared;  // [wave][row][token]
  const uint32_t lane = threadIdx.x & 63, wave = mx_wave(), q = lane / 16, r = lane % 16;
  const uint32_t steps = mx_steps(p.H), hsteps = mx_steps(p.F), blocks = hsteps * 4;
  const uint32_t first = blockIdx.x / blocks, f0 = blockIdx.x % blocks * 32;
  const uint32_t e = (uint32_t)ids[first];
  if (e >= p.E) return;
  const bool mine = threadIdx.x < A && (uint32_t)ids[threadIdx.x] == e;
  const uint64_t row = (uint64_t)e * p.F + f0, rest = (uint64_t)p.E * p.F - min(row, (uint64_t)p.E * p.F);
  const __amdgpu_buffer_rsrc_t g = mx_buffer(p.gc + row * steps * 64, rest * steps * 64);
  const __amdgpu_buffer_rsrc_t u = mx_buffer(p.uc + row * steps * 64, rest * steps * 64);
  const __amdgpu_buffer_rsrc_t gs = mx_buffer(p.gs + row * steps * 4, rest * steps * 4);
  const __amdgpu_buffer_rsrc_t us = mx_buffer(p.us + row * steps * 4, rest * steps * 4);
  // The members, in order; an earlier one: its work-group has this expert.
  const uint64_t ballot = __ballot(mine);
  if (lane == 0) counts[wave] = (uint32_t)__popcll(ballot);
  if (__syncthreads_or(mine && threadIdx.x < first)) return;
  uint32_t n = 0, at = lanes_below(ballot);
  for (uint32_t v = 0; v < 4; v++) {
    if (v < wave) at += counts[v];
    n += counts[v];
  }
  if (mine) member[at] = (uint16_t)threadIdx.x;
  for (uint32_t m0 = 0; m0 < n; m0 += kTok) {
    const uint32_t nm = min(n - m0, kTok);
    mx_f4 acc[4];
#pragma unroll
    for (int i = 0; i < 4; i++) acc[i] = mx_f4{0, 0, 0, 0};
    for (uint32_t s0 = 0; s0 < steps; s0 += kSteps) {
      const uint32_t ns = min(steps - s0, (uint32_t)kSteps);
      __syncthreads();  // (member; the LDS of the pass before)
      if (m0 == 0 || steps > kSteps) {
        // A row a load (or two): wave w has 16 rows, of gate or of up.
#pragma unroll 4
        for (uint32_t i = 0; i < 16; i++) {
          const uint32_t lr = wave * 16 + i, from = (lr % 32 * steps + s0) * 64;
#pragma unroll
          for (uint32_t j = 0; j < (kPitch + 1023) / 1024; j++) {
            const uint32_t piece = j * 64 + lane;
            if (piece < kPitch / 16 && piece < (ns + 3) / 4 * 16)
              lds_dma16(wave < 2 ? g : u, from + min((piece ^ (lr % 16)) * 16, ns * 64 - 16), wc + lr * kPitch + j * 1024);
          }
        }
        for (uint32_t i = wave % 2 * 64; i < 32 * ns; i += 128) {  // two waves gate's words, two up's
          const uint32_t lr = (i + lane) / ns, word = (i + lane) - lr * ns;
          if (i + lane < 32 * ns) lds_dma4(wave < 2 ? gs : us, (lr * steps + s0 + word) * 4, wsc + (wave < 2 ? 0 : 32 * ns) + i);
        }
      }
      for (uint32_t i = threadIdx.x; i < nm * ns * 16; i += 256) {
        const uint32_t xr = i / (ns * 16), gr = i - xr * (ns * 16);
        float v[8];
        load8<kX>(x + member[m0 + xr] / p.K * stride, (s0 * 16 + gr) * 8, p.H, v);
        uint32_t s;
        *(uint32_t *)(xc + xr * kXPitch + gr * 4) = mx_quantize8(v, s);
        if (gr % 4 == 0) ((uint8_t *)xsc)[xr * kSteps * 4 + gr / 4] = (uint8_t)s;
      }
      dma_barrier();
      const uint32_t xr = min(r, nm - 1);
      for (uint32_t k = wave; k < ns; k += 4) {
        const mx_i4 b = *(const mx_i4 *)(xc + xr * kXPitch + k * 64 + q * 16);
        const uint32_t sb = xsc[xr * kSteps + k] >> (8 * q);
#pragma unroll
        for (uint32_t i = 0; i < 4; i++) {
          const mx_i4 a = *(const mx_i4 *)(wc + (16 * i + r) * kPitch + ((4 * k + q) ^ r) * 16);
          acc[i] = mx_mfma16<0, 0>(a, b, acc[i], wsc[(16 * i + r) * ns + k] >> (8 * q), sb);
        }
      }
    }
    __syncthreads();  // (x's rows are read)
    if (r < kTok)
#pragma unroll
      for (uint32_t i = 0; i < 4; i++)
#pragma unroll
        for (uint32_t j = 0; j < 4; j++) sums[(wave * 64 + 16 * i + 4 * q + j) * kTok + r] = acc[i][j];
    __syncthreads();
    const uint32_t col = threadIdx.x % 32, t = threadIdx.x / 32;
    float gv = 0.0f, uv = 0.0f;
#pragma unroll
    for (uint32_t v = 0; v < 4; v++) gv += sums[(v * 64 + col) * kTok + t], uv += sums[(v * 64 + 32 + col) * kTok + t];
    h[t][col] = f0 + col < p.F ? mx_swiglu(gv, uv, p.limit) : 0.0f;
    __syncthreads();
    if (threadIdx.x < 4 * nm) {
      const uint32_t m = threadIdx.x / 4, part = threadIdx.x % 4;
      float v[8];
#pragma unroll
      for (int j = 0; j < 8; j++) v[j] = h[m][8 * part + j];
      uint32_t s;
      const uint32_t c = mx_quantize8(v, s);
      const uint64_t to = (uint64_t)member[m0 + m] * hsteps * 4 + f0 / 32;
      *(uint32_t *)(hc + to * 16 + part * 4) = c;
      if (part == 0) hs[to] = (uint8_t)s;
    }
  }
}

// A work-group: 16 rows of down for all assignments, and y's 16 columns. A wave takes every eighth of the experts that are
// used (its assignments 16 at a time), four steps of 128 a load, two loads of its own on their way.
constexpr uint32_t kFewHq = 56 * 1024;  // the assignments' rows of h in LDS

template <uint32_t kType>
__global__ void __launch_bounds__(512) mx4_down_few(MxExperts p, const uint8_t *hc, const uint8_t *hs, const int32_t *ids,
                                                    const float *w, uint32_t ntok, typename Elem<kType>::T *y, uint64_t stride) {
  struct Slot {
    alignas(16) uint8_t c[16 * 256];  // 16 rows, their 16-byte pieces exchanged by the row
    uint32_t s[16 * 4];
  };
  __shared__ Slot slot0[8];
  __shared__ Slot slot1[8];
  __shared__ __align__(16) uint8_t hq[kFewHq];
  __shared__ __align__(16) float o[kFew * 16];
  __shared__ uint32_t first[512];
  __shared__ uint16_t id[kFew], used[kFew], member[8][kFew];
  __shared__ uint32_t counts[8];
  const uint32_t lane = threadIdx.x & 63, wave = mx_wave(), q = lane / 16, r = lane % 16, A = ntok * p.K;
  const uint32_t steps = mx_steps(p.F), r0 = blockIdx.x * 16, pitch = steps * 64 + 16;
  uint32_t *hsc = (uint32_t *)(hq + A * pitch);  // [assignment][step]
  first[threadIdx.x] = ~0u;
  uint32_t e = p.E;
  if (threadIdx.x < A) {
    e = min((uint32_t)ids[threadIdx.x], p.E);
    id[threadIdx.x] = (uint16_t)e;
  }
  __syncthreads();
  if (e < p.E) atomicMin(first + e, threadIdx.x);
  __syncthreads();
  const bool owner = e < p.E && first[e] == threadIdx.x;
  const uint64_t ballot = __ballot(owner);
  if (lane == 0) counts[wave] = (uint32_t)__popcll(ballot);
  __syncthreads();
  uint32_t n = 0, at = lanes_below(ballot);
  for (uint32_t v = 0; v < 8; v++) {
    if (v < wave) at += counts[v];
    n += counts[v];
  }
  if (owner) used[at] = (uint16_t)threadIdx.x;
  __syncthreads();
  const uint32_t chunks = (steps + 3) / 4, units = wave < n ? ((n - 1 - wave) / 8 + 1) * chunks : 0;
  const uint32_t dr = lane / 16;  // (a load's rows: 4 j + dr)
  const auto load = [&](Slot &s, uint32_t unit) {
    const uint32_t ex = (uint32_t)__builtin_amdgcn_readfirstlane(id[used[wave + unit / chunks * 8]]), k = unit % chunks * 4;
    const uint32_t ns = min(steps - k, 4u);
    const uint64_t row = (uint64_t)ex * p.H + r0, rest = (uint64_t)p.E * p.H - row;
    const __amdgpu_buffer_rsrc_t c = mx_buffer(p.dc + row * steps * 64, rest * steps * 64);
    const __amdgpu_buffer_rsrc_t sc = mx_buffer(p.ds + row * steps * 4, rest * steps * 4);
#pragma unroll
    for (uint32_t j = 0; j < 4; j++) {
      const uint32_t lr = 4 * j + dr;
      lds_dma16(c, (lr * steps + k) * 64 + min(((lane % 16) ^ lr) * 16, ns * 64 - 16), s.c + j * 1024);
    }
    lds_dma4(sc, (lane / 4 * steps + k + min(lane % 4, ns - 1)) * 4, s.s);
  };
  if (units > 0) load(slot0[wave], 0);
  if (units > 1) load(slot1[wave], 1);
  for (uint32_t i = threadIdx.x; i < A * steps * 4; i += 512) {
    const uint32_t a = i / (steps * 4), piece = i - a * (steps * 4);
    *(uint4 *)(hq + a * pitch + piece * 16) = ((const uint4 *)hc)[i];
  }
  for (uint32_t i = threadIdx.x; i < A * steps; i += 512) hsc[i] = ((const uint32_t *)hs)[i];
  __syncthreads();
  uint32_t nm = 0;
  const auto use = [&](const Slot &s, uint32_t unit, bool more) {
    // This unit's load has arrived; the next one's five may be outstanding.
    asm volatile("" ::: "memory");
    if (more)
      __builtin_amdgcn_s_waitcnt(0x0f75);
    else
      __builtin_amdgcn_s_waitcnt(0x0f70);
    asm volatile("" ::: "memory");
    const uint32_t k = unit % chunks * 4, ns = min(steps - k, 4u);
    if (k == 0) {  // the expert's assignments
      const uint32_t ex = id[used[wave + unit / chunks * 8]];
      nm = 0;
      for (uint32_t a0 = 0; a0 < A; a0 += 64) {
        const bool is = a0 + lane < A && id[a0 + lane] == ex;
        const uint64_t bal = __ballot(is);
        if (is) member[wave][nm + lanes_below(bal)] = (uint16_t)(a0 + lane);
        nm += (uint32_t)__popcll(bal);
      }
      __builtin_amdgcn_s_waitcnt(0xc07f);
      __builtin_amdgcn_wave_barrier();
    }
    mx_i4 a[4];
    uint32_t sa[4];
#pragma unroll
    for (uint32_t j = 0; j < 4; j++) {
      a[j] = *(const mx_i4 *)(s.c + r * 256 + ((4 * j + q) ^ r) * 16);
      sa[j] = s.s[r * 4 + j] >> (8 * q);
    }
    for (uint32_t m0 = 0; m0 < nm; m0 += 16) {
      const uint32_t as = member[wave][min(m0 + r, nm - 1)];
      mx_f4 c = {0, 0, 0, 0};
      float4 *to = (float4 *)(o + as * 16 + 4 * q);
      if (k != 0) {
        const float4 v = *to;
        c = mx_f4{v.x, v.y, v.z, v.w};
      }
#pragma unroll
      for (uint32_t j = 0; j < 4; j++) {
        if (j >= ns) break;
        const mx_i4 b = *(const mx_i4 *)(hq + as * pitch + (k + j) * 64 + q * 16);
        c = mx_mfma16<0, 0>(a[j], b, c, sa[j], hsc[as * steps + k + j] >> (8 * q));
      }
      if (m0 + r < nm) *to = make_float4(c[0], c[1], c[2], c[3]);
    }
  };
  for (uint32_t i = 0; i < units; i += 2) {
    use(slot0[wave], i, i + 1 < units);
    if (i + 2 < units) load(slot0[wave], i + 2);
    if (i + 1 >= units) break;
    use(slot1[wave], i + 1, i + 2 < units);
    if (i + 3 < units) load(slot1[wave], i + 3);
  }
  __syncthreads();
  for (uint32_t i = threadIdx.x; i < ntok * 16; i += 512) {
    const uint32_t t = i / 16, c = i % 16;
    float s = 0.0f;
    for (uint32_t k = 0; k < p.K; k++)
      if (id[t * p.K + k] < p.E) s += w[t * p.K + k] * o[(t * p.K + k) * 16 + c];
    if (r0 + c < p.H) y[(uint64_t)t * stride + r0 + c] = (typename Elem<kType>::T)s;
  }
}

// y's columns c0 .. c0 + cols (a multiple of 4 wide; H ends them) from the assignments' sums, `cols` apart, each token's in
// rank order: four columns a thread, all ranks' sums loaded before the first is added.
template <uint32_t kType>
__global__ void __launch_bounds__(256) mx4_combine(const float *o, const int32_t *ids, const float *w, uint32_t ntok, uint32_t E,
                                                   uint32_t K, uint32_t H, uint32_t c0, uint32_t cols,
                                                   typename Elem<kType>::T *y, uint64_t stride) {
  typedef typename Elem<kType>::T T;
  const uint32_t per = cols / 4;  // threads a token
  const uint64_t i = (uint64_t)blockIdx.x * 256 + threadIdx.x;
  const uint64_t t = i / per;
  const uint32_t c = (uint32_t)(i - t * per) * 4;
  if (t >= ntok || c0 + c >= H) return;
  float4 s = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  const float *from = o + t * K * cols + c;
#pragma unroll
  for (uint32_t k0 = 0; k0 < 16; k0 += 8) {
    float4 v[8];
    float f[8];
#pragma unroll
    for (uint32_t k = 0; k < 8; k++) {
      const bool on = k0 + k < K && (uint32_t)ids[t * K + min(k0 + k, K - 1)] < E;
      f[k] = on ? w[t * K + k0 + k] : 0.0f;
      v[k] = on ? *(const float4 *)(from + (uint64_t)(k0 + k) * cols) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    }
#pragma unroll
    for (uint32_t k = 0; k < 8; k++)
      s.x += f[k] * v[k].x, s.y += f[k] * v[k].y, s.z += f[k] * v[k].z, s.w += f[k] * v[k].w;
    if (K <= 8) break;
  }
  T *to = y + t * stride + c0 + c;
  const T e[4] = {(T)s.x, (T)s.y, (T)s.z, (T)s.w};
  if (c0 + c + 4 <= H) {
    struct __attribute__((packed)) Four {
      T e[4];
    };
    *(Four *)to = Four{{e[0], e[1], e[2], e[3]}};
  } else {
    for (uint32_t j = 0; c0 + c + j < H; j++) to[j] = e[j];
  }
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

// How a call runs. Few assignments, whose rows of h fit LDS, without sorting them: up to 96 (8 tokens of 10 of 512 experts 41
// us, sorted 45; 12 of 64 experts' 10: 35 us, sorted 32), or to kFew where they are of few experts (32 tokens of 4 of 16
// experts 21 us, sorted 25). n_embd 2048, n_ff 512 here and below.
constexpr uint64_t kChunkBytes = 256 << 20;

struct Plan {
  uint32_t A, rows, pitch, chunk, max_tiles;
  bool few;
  uint64_t xc, xs, hc, hs, o, order, tiles, n_tiles, bytes;  // the work buffer's parts

  Plan(const moe_mx4_experts &e, uint32_t T) {
    A = T * e.n_used;
    few = A <= (e.n_expert <= 32 ? kFew : 96) && A * (mx_steps(e.n_ff) * 68 + 16) <= kFewHq;
    // Tiles of 32, 64 or 128 positions: the more an expert has on average, the fewer times its weights are read. 301 tokens
    // of 10 of 512 experts (6 each) 181, 191 and 243 us; 2048 (40) 290, 261 and 302; 4096 (80) 430, 397 and 374, with skewed
    // experts 463, 416 and 436; 1024 of 8 of 128 (64) 97, 88 and 92; 4096 of 4 of 16 (1024) 131, 112 and 113.
    const uint32_t mean = A / e.n_expert;
    rows = mean < 24 ? 32 : mean < 96 ? 64 : 128;
    pitch = (e.n_embd + 255) / 256 * 256;
    // The sums of all assignments at once, or of as many columns at a time as 256 MB hold, about the last-level cache (4096
    // tokens of 10 experts: 335 MB of sums, 304 us; 96 MB at a time 312, all at once 303, but up to 17 GB of work).
    // (few: there are no such sums, and A may be 0.)
    chunk = few ? pitch : std::min<uint64_t>(pitch, std::max<uint64_t>(256, kChunkBytes / (4ull * A) / 256 * 256));
    max_tiles = std::min(A, e.n_expert + A / rows);
    uint64_t at = 0;
    const auto part = [&](uint64_t n) {
      const uint64_t was = at;
      at += (n + 255) / 256 * 256;
      return was;
    };
    xc = part(few ? 0 : moe_mx4_code_bytes(T, e.n_embd)), xs = part(few ? 0 : moe_mx4_scale_bytes(T, e.n_embd));
    hc = part(moe_mx4_code_bytes(A, e.n_ff)), hs = part(moe_mx4_scale_bytes(A, e.n_ff));
    o = part(few ? 0 : (uint64_t)A * chunk * 4);
    order = part(few ? 0 : (uint64_t)A * 4);
    tiles = part(few ? 0 : (uint64_t)max_tiles * sizeof(MoeTile)), n_tiles = part(few ? 0 : 4);
    bytes = at;
  }
};

}  // namespace

extern "C" {

MOE_API uint64_t moe_mx4_experts_work_bytes(const moe_mx4_experts *e, uint32_t ntok) {
  uint64_t n = 0;
  (void)op_guarded([&] {
    check_experts(e, ntok);
    n = Plan(*e, ntok).bytes;
  });
  return n;
}

MOE_API moe_status moe_mx4_experts_async(const moe_mx4_experts *e, const void *x, uint64_t x_stride, uint32_t ntok,
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
    const MxExperts p{e->gate.codes, e->gate.scales, e->up.codes, e->up.scales, e->down.codes, e->down.scales, E, K, H, F,
                      e->swiglu_limit};
    const uint8_t *xc = b + at.xc, *xs = b + at.xs;
    uint8_t *hc = b + at.hc, *hs = b + at.hs;
    float *o = (float *)(b + at.o);
    if (at.few) {
      op_by_type(e->x_type, [&](auto t) {
        constexpr uint32_t kX = decltype(t)::value;
        const auto run = [&](auto kernel) {
          op_launch(kernel, (uint64_t)A * mx_steps(F) * 4, 256, stream, p, (const typename Elem<kX>::T *)x, x_stride, ids, A, hc, hs);
        };
        if (mx_steps(H) <= 16)
          run(mx4_gate_up_few<kX, 16>);
        else
          run(mx4_gate_up_few<kX, 24>);
      });
      op_by_type(e->y_type, [&](auto t) {
        constexpr uint32_t kY = decltype(t)::value;
        op_launch(mx4_down_few<kY>, (H + 15) / 16, 512, stream, p, (const uint8_t *)hc, (const uint8_t *)hs, ids, w, ntok,
                  (typename Elem<kY>::T *)y, y_stride);
      });
      return;
    }
    const auto combine = [&](uint32_t c0, uint32_t cols) {
      const uint64_t n = ((uint64_t)ntok * (cols / 4) + 255) / 256;
      const auto run = [&](auto kernel, auto *to) {
        op_launch(kernel, n, 256, stream, (const float *)o, ids, w, ntok, E, K, H, c0, cols, to, y_stride);
      };
      if (e->y_type == QT_F32) run(mx4_combine<QT_F32>, (float *)y);
      if (e->y_type == QT_F16) run(mx4_combine<QT_F16>, (_Float16 *)y);
      if (e->y_type == QT_BF16) run(mx4_combine<QT_BF16>, (__bf16 *)y);
    };
    uint32_t *order = (uint32_t *)(b + at.order), *nt = (uint32_t *)(b + at.n_tiles);
    MoeTile *tiles = (MoeTile *)(b + at.tiles);
    op_by_type(e->x_type, [&](auto t) {
      constexpr uint32_t kX = decltype(t)::value;
      const uint32_t slices = (A + kSlice - 1) / kSlice, groups = ntok * mx_steps(H) * 16;
      op_launch(mx4_prepare<kX>, slices + (groups + kGroups - 1) / kGroups, 1024, stream, ids, A, E, slices, at.rows, order,
                tiles, nt, (const typename Elem<kX>::T *)x, x_stride, ntok, H, b + at.xc, b + at.xs);
    });
    const auto run = [&](auto gate_up, auto down, uint32_t bn) {
      op_launch(gate_up, item_blocks((uint64_t)at.max_tiles * (mx_steps(F) * 256 / bn), mx_steps(F) * 256 / bn), 256, stream, p, xc, xs, ntok,
                (const uint32_t *)order, (const MoeTile *)tiles, (const uint32_t *)nt, hc, hs);
      for (uint32_t c = 0; c < at.pitch; c += at.chunk) {
        const uint32_t cols = std::min(at.chunk, at.pitch - c);
        op_launch(down, item_blocks((uint64_t)at.max_tiles * (cols / bn), cols / bn), 256, stream, p, (const uint8_t *)hc,
                  (const uint8_t *)hs, A, (const uint32_t *)order, (const MoeTile *)tiles, (const uint32_t *)nt, c, cols, o);
        combine(c, cols);
      }
    };
    if (at.rows == 32) run(mx4_gate_up_tiles<1, 1>, mx4_down_tiles<1, 1>, 256);
    if (at.rows == 64) run(mx4_gate_up_tiles<1, 2>, mx4_down_tiles<1, 2>, 128);
    if (at.rows == 128) run(mx4_gate_up_tiles<2, 2>, mx4_down_tiles<2, 2>, 128);
  });
}

}  // extern "C"
