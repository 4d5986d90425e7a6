// The experts of routed tokens in MX4 (moe_mx4_experts_async).
//
// Many tokens: the assignments (token * n_used + rank) are sorted by expert and cut into MoeTiles of kRows positions;
// gate and up of a tile are one product whose epilogue applies the SwiGLU and quantises h, 32 neighbours of a row being in
// one wave's registers; down follows on the positions' rows, its sums go to the assignments' rows, and a last kernel adds
// each token's in rank order. Bound by reading the experts' weights (once for all of a tile's tokens) until an expert has
// some hundreds of tokens.
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

// ---- the assignments by expert

constexpr uint32_t kSlice = 4096;  // ids a work-group sorts

// How often each expert is in each slice.
__global__ void __launch_bounds__(1024) mx4_count(const int32_t *ids, uint32_t A, uint32_t E, uint32_t *counts) {
  __shared__ uint32_t n[512];
  if (threadIdx.x < 512) n[threadIdx.x] = 0;
  __syncthreads();
  const uint32_t end = min(A, (blockIdx.x + 1) * kSlice);
  for (uint32_t i = blockIdx.x * kSlice + threadIdx.x; i < end; i += 1024) {
    const uint32_t e = (uint32_t)ids[i];
    if (e < E) atomicAdd(n + e, 1u);
  }
  __syncthreads();
  if (threadIdx.x < E) counts[blockIdx.x * E + threadIdx.x] = n[threadIdx.x];
}

// The inclusive sums of v over the work-group's 1024 threads in steps of 512 values: thread e's own (e < 512).
__device__ __forceinline__ uint32_t scan512(uint32_t v, uint32_t *lds) {
  const uint32_t e = threadIdx.x;
  __syncthreads();
  if (e < 512) lds[e] = v;
  for (uint32_t d = 1; d < 512; d *= 2) {
    __syncthreads();
    const uint32_t add = e < 512 && e >= d ? lds[e - d] : 0;
    __syncthreads();
    if (e < 512) lds[e] += add;
  }
  __syncthreads();
  return e < 512 ? lds[e] : 0;
}

// A slice's assignments to their places (order[place] = assignment; within an expert by slice), and, by the first
// work-group, the tiles of at most `rows` places each. With one slice the counts are taken here.
__global__ void __launch_bounds__(1024) mx4_place(const int32_t *ids, uint32_t A, uint32_t E, const uint32_t *counts,
                                                  uint32_t rows, uint32_t *order, MoeTile *tiles, uint32_t *n_tiles) {
  __shared__ uint32_t next[512];
  __shared__ uint32_t lds[512];
  const uint32_t e = threadIdx.x, first = blockIdx.x * kSlice, end = min(A, first + kSlice);
  uint32_t all = 0, before = 0;  // expert e's assignments, those of the slices before this one
  if (gridDim.x == 1) {
    if (e < 512) next[e] = 0;
    __syncthreads();
    for (uint32_t i = e; i < end; i += 1024)
      if ((uint32_t)ids[i] < E) atomicAdd(next + (uint32_t)ids[i], 1u);
    __syncthreads();
    all = e < E ? next[e] : 0;
  } else if (e < E) {
    for (uint32_t b = 0; b < gridDim.x; b++) {
      const uint32_t n = counts[b * E + e];
      all += n, before += b < blockIdx.x ? n : 0;
    }
  }
  const uint32_t start = scan512(all, lds) - all;
  if (blockIdx.x == 0) {
    const uint32_t n = (all + rows - 1) / rows, last = scan512(n, lds);
    if (e < E)
      for (uint32_t j = 0; j < n; j++) tiles[last - n + j] = MoeTile{e, e, start + j * rows, min(rows, all - j * rows)};
    if (e == 511) *n_tiles = last;
  }
  __syncthreads();
  if (e < 512) next[e] = start + before;
  __syncthreads();
  for (uint32_t i = first + e; i < end; i += 1024) {
    const uint32_t id = (uint32_t)ids[i];
    if (id < E) order[atomicAdd(next + id, 1u)] = i;
  }
}

// ---- the products

struct MxExperts {
  const uint8_t *gc, *gs, *uc, *us, *dc, *ds;
  uint32_t E, K, H, F;
  float limit;
};

// A launch's work-groups to its items (parts a tile) so that an XCD (work-groups go to the eight in turn) has runs of four
// tiles: an expert's tiles share its weights in that L2, while the experts with one tile are dealt over all of them (whole
// eighths of the list on an XCD left most of the distinct weights to a few: 4096 skewed tokens 132 us instead of the
// figures below). ~0: none.
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
__global__ void __launch_bounds__(256, TM == 1 && WM == 2 ? 3 : 2) mx4_gate_up_tiles(MxExperts p, const uint8_t *xc, const uint8_t *xs, uint32_t ntok,
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
  c.clear();
  c.run(
      s0, s1, scales, stages,
      [&](typename Tile::Stage &s, uint32_t k) { g.load(k, s.w), u.load(k, s.w + kCols * 128), x.load(k, s.x); },
      [&](typename Tile::Scales &s, uint32_t k) {
        g.load_scales(k, s.w), u.load_scales(k, s.w + kCols * mx_pitch(k, steps)), x.load_scales(k, s.x);
      },
      [&](uint32_t k) { return mx_pitch(k, steps); }, [&](uint32_t k) { return min(steps - 2 * k, 2u); }, [](uint32_t) {});
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

// An item: a tile and a few times BN of the `cols` rows of down from r0 on, one after the other on the same pipeline, so many
// that the launch has about 2048 items. Writes the sums to the assignments' rows of o, `cols` apart (a multiple of 256): a
// lane has a column of 16 rows, so that a store is of whole lines (two rows of 32 columns; with a row's four neighbours a
// lane it was 32 rows of 32 bytes: 4096 tokens 172 us in all, now see below).
template <int TM, int WM>
__global__ void __launch_bounds__(256, TM == 1 && WM == 2 ? 3 : 2) mx4_down_tiles(MxExperts p, const uint8_t *hc, const uint8_t *hs, uint32_t A,
                                                      const uint32_t *order, const MoeTile *tiles, const uint32_t *n_tiles,
                                                      uint32_t r0, uint32_t cols, float *o) {
  typedef MxTile<TM, 2, WM, true, true> Tile;
  __shared__ typename Tile::Stage s0;
  __shared__ typename Tile::Stage s1;
  __shared__ typename Tile::Scales scales;
  __shared__ __align__(16) uint32_t place[Tile::BM];  // where a row of the tile goes, in bytes
  constexpr uint32_t kNowhere = 0xf0000000u;           // (out of the buffer: a store there is dropped)
  const uint32_t steps = mx_steps(p.F), total = cols / Tile::BN, nt = *n_tiles;
  const uint32_t blocks = min(max(nt * total / 2048, 1u), total), parts = (total + blocks - 1) / blocks;
  const uint32_t item = item_of(nt * parts, parts);
  if (item == ~0u) return;
  const MoeTile tile = tiles[item / parts];
  const uint32_t b0 = item % parts * blocks, nb = min(blocks, total - b0);
  const uint32_t stages = (steps + 3) / 4 * 2;  // of BN rows: whole pairs (the last one may be empty)
  const uint64_t row = (uint64_t)tile.expert * p.H + r0 + b0 * Tile::BN, rest = (uint64_t)p.E * p.H - min(row, (uint64_t)p.E * p.H);
  const auto same = [](uint32_t r) { return r; };
  const MxSource<Tile::BM> x(hc, hs, A, steps, [&](uint32_t r) { return tile.start + min(r, tile.count - 1); });
  const MxSource<Tile::BN> w(p.dc + row * steps * 64, p.ds + row * steps * 4, rest, steps, same);
  const uint32_t lane = threadIdx.x & 63, q = lane / 32;
  if (threadIdx.x < Tile::BM)
    place[threadIdx.x] = threadIdx.x < tile.count ? order[tile.start + threadIdx.x] * cols * 4 : kNowhere;
  const __amdgpu_buffer_rsrc_t to = mx_buffer((const uint8_t *)o, (uint64_t)A * cols * 4);
  const uint32_t col = (b0 * Tile::BN + Tile::w_row() + lane % 32) * 4;
  Tile c;
  c.clear();
  const auto store = [&](uint32_t n) {  // the sums of the n-th BN rows
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
            __builtin_amdgcn_raw_buffer_store_b32(__float_as_uint(c.acc[f][m][4 * j + i]), to, at[i] + col,
                                                  (n * Tile::BN + f * Tile::kStep) * 4, 0);
      }
    c.clear();
  };
  c.run(
      s0, s1, scales, nb * stages,
      [&](typename Tile::Stage &s, uint32_t i) {
        const uint32_t n = i / stages, k = i - n * stages;
        if (2 * k < steps) w.load(k, s.w, n * Tile::BN), x.load(k, s.x);
      },
      [&](typename Tile::Scales &s, uint32_t i) {
        const uint32_t n = i / stages, k = i - n * stages;
        w.load_scales(k, s.w, n * Tile::BN), x.load_scales(k, s.x);
      },
      [&](uint32_t i) { return mx_pitch(i % stages, steps); },
      [&](uint32_t i) { return min(steps - min(2 * (i % stages), steps), 2u); },
      [&](uint32_t i) {
        if (i % stages == stages - 1) store(i / stages);
      });
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
                                               float *o, uint32_t pitch) {
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
      if (r0 + 4 * q + i < H) o[(uint64_t)a * pitch + r0 + 4 * q + i] = c[i];
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

// How a call runs: assignments at most kFew: without sorting them.
constexpr uint32_t kFew = 256;
constexpr uint64_t kChunkBytes = 96 << 20;

struct Plan {
  uint32_t A, rows, slices, pitch, chunk, max_tiles;
  bool few;
  uint64_t xc, xs, h, hc, hs, o, counts, order, tiles, n_tiles, bytes;  // the work buffer's parts

  Plan(const moe_mx4_experts &e, uint32_t T) {
    A = T * e.n_used, few = A <= kFew;
    // Tiles of 32, 64 or 128 positions: the more an expert has on average, the fewer times its weights are read.
    const uint32_t mean = A / e.n_expert;
    rows = mean < 24 ? 32 : mean < 96 ? 64 : 128;
    slices = (A + kSlice - 1) / kSlice;
    pitch = (e.n_embd + 255) / 256 * 256;
    // The sums of all assignments at once, or of a part of the columns at a time that the last-level cache (256 MB) keeps
    // until they are added.
    chunk = few ? pitch : std::min<uint64_t>(pitch, std::max<uint64_t>(256, kChunkBytes / (4ull * A) / 256 * 256));
    max_tiles = std::min(A, e.n_expert + A / rows);
    uint64_t at = 0;
    const auto part = [&](uint64_t n) {
      const uint64_t was = at;
      at += (n + 255) / 256 * 256;
      return was;
    };
    xc = part(moe_mx4_code_bytes(T, e.n_embd)), xs = part(moe_mx4_scale_bytes(T, e.n_embd));
    h = part(few ? (uint64_t)A * e.n_ff * 4 : 0);
    hc = part(moe_mx4_code_bytes(A, e.n_ff)), hs = part(moe_mx4_scale_bytes(A, e.n_ff));
    o = part((uint64_t)A * chunk * 4);
    counts = part(few ? 0 : (uint64_t)slices * e.n_expert * 4), order = part(few ? 0 : (uint64_t)A * 4);
    tiles = part(few ? 0 : (uint64_t)max_tiles * sizeof(MoeTile)), n_tiles = part(4);
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
    op_rows(x, x_stride, H, e->x_type);
    op_rows(y, y_stride, H, e->y_type);
    op_require(ids && w && op_aligned(ids, 4) && op_aligned(w, 4), "null or misaligned ids or w");
    const Plan at(*e, ntok);
    op_work(work, work_bytes, at.bytes);
    if (!ntok) return;
    OnDevice on(e->device);
    uint8_t *b = (uint8_t *)work;
    mx4_quantize_launch(e->x_type, x, x_stride, moe_mx4_matrix{b + at.xc, b + at.xs, ntok, H}, stream);
    const MxExperts p{e->gate.codes, e->gate.scales, e->up.codes, e->up.scales, e->down.codes, e->down.scales, E, K, H, F,
                      e->swiglu_limit};
    const uint8_t *xc = b + at.xc, *xs = b + at.xs;
    uint8_t *hc = b + at.hc, *hs = b + at.hs;
    float *o = (float *)(b + at.o);
    const auto combine = [&](uint32_t c0, uint32_t cols) {
      const uint64_t n = ((uint64_t)ntok * (cols / 4) + 255) / 256;
      const auto run = [&](auto kernel, auto *to) {
        op_launch(kernel, n, 256, stream, (const float *)o, ids, w, ntok, E, K, H, c0, cols, to, y_stride);
      };
      if (e->y_type == QT_F32) run(mx4_combine<QT_F32>, (float *)y);
      if (e->y_type == QT_F16) run(mx4_combine<QT_F16>, (_Float16 *)y);
      if (e->y_type == QT_BF16) run(mx4_combine<QT_BF16>, (__bf16 *)y);
    };
    if (at.few) {
      op_launch(mx4_gate_up, (uint64_t)A * ((F + 15) / 16), 64, stream, xc, xs, p.gc, p.gs, p.uc, p.us, ids, E, K, H, F,
                e->swiglu_limit, (float *)(b + at.h));
      mx4_quantize_launch(QT_F32, b + at.h, F, moe_mx4_matrix{hc, hs, A, F}, stream);
      op_launch(mx4_down, (uint64_t)A * ((H + 15) / 16), 64, stream, (const uint8_t *)hc, (const uint8_t *)hs, p.dc, p.ds,
                ids, E, H, F, o, at.pitch);
      return combine(0, at.pitch);
    }
    uint32_t *counts = (uint32_t *)(b + at.counts), *order = (uint32_t *)(b + at.order), *nt = (uint32_t *)(b + at.n_tiles);
    MoeTile *tiles = (MoeTile *)(b + at.tiles);
    if (at.slices > 1) op_launch(mx4_count, at.slices, 1024, stream, ids, A, E, counts);
    op_launch(mx4_place, at.slices, 1024, stream, ids, A, E, (const uint32_t *)counts, at.rows, order, tiles, nt);
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
