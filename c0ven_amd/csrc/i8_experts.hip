// The experts of routed tokens in I8 (moe_i8_experts_async).
//
// Many tokens: the assignments are sorted by expert and cut into MoeTiles; x's rows are quantised; gate and up of a tile are one
// product whose epilogue applies the SwiGLU; the rows of h (fp32: a row's scale needs all of it) are quantised; down follows, its
// values in fp32 by position, and each token's are summed in rank order.
#include "../../include/c0ven_moe_tile.h"
#include "dispatch.h"
#include "experts.h"
#include "i8_api.h"
#include "i8_few.h"
#include "i8_gemm.h"

#include <algorithm>

namespace c0ven {

struct I8Experts {
  const int8_t *gc, *uc, *dc;
  const float *gs, *us, *ds;
  uint32_t E, K, H, F;
  float limit;
};

// An item: a tile and 32 WN columns of h (their rows of gate and of up). Writes the positions' rows of h, `pitch` apart: a lane
// has a column of 16 rows, so that a store is of whole lines.
template <int TM, int WM>
__global__ void __launch_bounds__(256) i8_gate_up_tiles(I8Experts p, const int8_t *xc, const float *xs, uint32_t ntok,
                                                        const int32_t *order, const MoeTile *tiles, const uint32_t *n_tiles,
                                                        float *h, uint32_t pitch) {
  typedef I8Tile<TM, 2, WM, true, true> Tile;
  constexpr uint32_t kCols = Tile::BN / 2;
  __shared__ typename Tile::X x0;
  __shared__ typename Tile::X x1;
  __shared__ typename Tile::W w0;
  __shared__ typename Tile::W w1;
  __shared__ __align__(16) float sx[Tile::BM];
  const uint32_t steps = i8_steps(p.H), parts = (p.F + kCols - 1) / kCols, item = item_of(*n_tiles * parts, parts);
  if (item == ~0u) return;
  const MoeTile tile = tiles[item / parts];
  const uint32_t f0 = item % parts * kCols;
  const uint64_t row = (uint64_t)tile.expert * p.F + f0, rest = (uint64_t)p.E * p.F - row;
  const auto same = [](uint32_t r) { return r; };
  const auto token = [&](uint32_t r) { return (uint32_t)order[tile.start + r] / p.K; };
  const I8Source<Tile::BM> x(xc, ntok, steps, [&](uint32_t r) { return r < tile.count ? token(r) : ntok; });
  const I8Source<kCols> g(p.gc + row * steps * kI8Row, rest, steps, same);
  const I8Source<kCols> u(p.uc + row * steps * kI8Row, rest, steps, same);
  if (threadIdx.x < Tile::BM) sx[threadIdx.x] = threadIdx.x < tile.count ? xs[token(threadIdx.x)] : 0.0f;
  Tile c;
  c.run2(
      x0, x1, w0, w1, steps, [&](typename Tile::X &s, uint32_t k) { x.load(k, s.b); },
      [&](typename Tile::W &s, uint32_t k) { g.load(k, s.b), u.load(k, s.b + kCols * kI8Row); });
  const uint32_t lane = threadIdx.x & 63, q = lane / 32, col = Tile::w_row() + lane % 32;
  const bool in = f0 + col < p.F;
  const float sg = in ? p.gs[row + col] : 0.0f, su = in ? p.us[row + col] : 0.0f;
  const __amdgpu_buffer_rsrc_t to =
      mx_buffer((const uint8_t *)(h + (uint64_t)tile.start * pitch), (uint64_t)tile.count * pitch * 4);
#pragma unroll
  for (int m = 0; m < TM; m++)
#pragma unroll
    for (int j = 0; j < 4; j++) {
      const uint32_t r = Tile::x_row() + 32 * m + 8 * j + 4 * q;
      const float4 v = *(const float4 *)(sx + r);
      const float s[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
      for (int i = 0; i < 4; i++) {
        const float gv = i8_value(c.acc[0][m][4 * j + i], s[i], sg), uv = i8_value(c.acc[1][m][4 * j + i], s[i], su);
        const uint32_t at = in ? ((r + i) * pitch + f0 + col) * 4 : kNowhere;
        __builtin_amdgcn_raw_buffer_store_b32(__float_as_uint(expert_swiglu(gv, uv, p.limit)), to, at, 0, 0);
      }
    }
}

// An item: a tile and BN of the `cols` rows of down from r0 on. Writes the positions' rows of o, `cols` apart (a multiple of 256).
template <int TM, int WM>
__global__ void __launch_bounds__(256) i8_down_tiles(I8Experts p, const int8_t *hc, const float *hs, const MoeTile *tiles,
                                                     const uint32_t *n_tiles, uint32_t r0, uint32_t cols, float *o) {
  typedef I8Tile<TM, 2, WM, true, true> Tile;
  __shared__ typename Tile::X x0;
  __shared__ typename Tile::X x1;
  __shared__ typename Tile::W w0;
  __shared__ typename Tile::W w1;
  __shared__ __align__(16) float sh[Tile::BM];
  const uint32_t steps = i8_steps(p.F), parts = cols / Tile::BN, item = item_of(*n_tiles * parts, parts);
  if (item == ~0u) return;
  const MoeTile tile = tiles[item / parts];
  const uint32_t c0 = item % parts * Tile::BN;
  const uint64_t all = (uint64_t)p.E * p.H, row = min((uint64_t)tile.expert * p.H + r0 + c0, all);
  const auto same = [](uint32_t r) { return r; };
  const I8Source<Tile::BM> x(hc + (uint64_t)tile.start * steps * kI8Row, tile.count, steps, same);
  const I8Source<Tile::BN> w(p.dc + row * steps * kI8Row, all - row, steps, same);
  if (threadIdx.x < Tile::BM) sh[threadIdx.x] = threadIdx.x < tile.count ? hs[tile.start + threadIdx.x] : 0.0f;
  Tile c;
  c.run2(
      x0, x1, w0, w1, steps, [&](typename Tile::X &s, uint32_t k) { x.load(k, s.b); },
      [&](typename Tile::W &s, uint32_t k) { w.load(k, s.b); });
  const uint32_t lane = threadIdx.x & 63, q = lane / 32, col = Tile::w_row() + lane % 32;
  float sd[2];
#pragma unroll
  for (int f = 0; f < 2; f++) sd[f] = row + col + f * Tile::kStep < all ? p.ds[row + col + f * Tile::kStep] : 0.0f;
  const __amdgpu_buffer_rsrc_t to = mx_buffer((const uint8_t *)(o + (uint64_t)tile.start * cols), (uint64_t)tile.count * cols * 4);
#pragma unroll
  for (int m = 0; m < TM; m++)
#pragma unroll
    for (int j = 0; j < 4; j++) {
      const uint32_t r = Tile::x_row() + 32 * m + 8 * j + 4 * q;
      const float4 v = *(const float4 *)(sh + r);
      const float s[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
      for (int i = 0; i < 4; i++)
#pragma unroll
        for (int f = 0; f < 2; f++)
          __builtin_amdgcn_raw_buffer_store_b32(__float_as_uint(i8_value(c.acc[f][m][4 * j + i], s[i], sd[f])), to,
                                                ((r + i) * cols + c0 + col) * 4, f * Tile::kStep * 4, 0);
    }
}

// ---- few assignments (at most kFew): no sorting, two launches. Bound by latency and by reading the experts' weights, which
// go to LDS as whole rows: all that a work-group needs is on its way at once.

constexpr uint32_t kFew = 160;

// A work-group: an expert and 16 columns of h, for the tokens that use the expert, kTok at a time: the assignment that is the
// first with its expert does the work, the others' work-groups leave. Quantises x itself (while the weights come) and writes the
// assignments' rows of h, `pitch` apart. Four waves share the k axis, kSteps steps of 128 at a time (all of n_embd, where it is
// not longer); the sums are joined in LDS.
template <uint32_t kX, int kSteps>
__global__ void __launch_bounds__(256) i8_gate_up_few(I8Experts p, const typename Elem<kX>::T *x, uint64_t stride,
                                                      const int32_t *ids, uint32_t A, float *h, uint32_t pitch) {
  constexpr uint32_t kTok = 6, kPitch = kSteps * kI8Row, kXPitch = kPitch + 16;
  static_assert(kSteps % 2 == 0, "rows of 16 pieces");
  __shared__ __align__(16) uint8_t wc[32 * kPitch];  // gate's 16 rows, up's; a row's 16-byte pieces exchanged by r % 16
  __shared__ __align__(16) uint8_t xc[kTok * kXPitch];
  __shared__ int sums[4][32][kTok];
  __shared__ uint32_t most[kTok];
  __shared__ uint16_t member[kFew];
  __shared__ uint32_t counts[4];
  const uint32_t lane = threadIdx.x & 63, wave = mx_wave(), q = lane / 16, r = lane % 16;
  const uint32_t steps = i8_steps(p.H), blocks = (p.F + 15) / 16;
  const uint32_t first = blockIdx.x / blocks, f0 = blockIdx.x % blocks * 16;
  const uint32_t e = (uint32_t)ids[first];
  if (e >= p.E) return;
  const bool mine = threadIdx.x < A && (uint32_t)ids[threadIdx.x] == e;
  const uint64_t row = (uint64_t)e * p.F + f0, rest = (uint64_t)p.E * p.F - row;
  const __amdgpu_buffer_rsrc_t w = mx_buffer((const uint8_t *)(wave < 2 ? p.gc : p.uc) + row * steps * kI8Row, rest * steps * kI8Row);
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
    mx_i4 acc[2] = {{0, 0, 0, 0}, {0, 0, 0, 0}};
    for (uint32_t s0 = 0; s0 < steps; s0 += kSteps) {
      const uint32_t ns = min(steps - s0, (uint32_t)kSteps);
      __syncthreads();  // (member; the LDS of the pass before)
      if (m0 == 0 || steps > kSteps) {
        // 64 pieces of a row a load: wave w has eight rows, of gate or of up.
#pragma unroll 4
        for (uint32_t i = 0; i < 8; i++) {
          const uint32_t lr = wave * 8 + i, from = (lr % 16 * steps + s0) * kI8Row;
#pragma unroll
          for (uint32_t j = 0; j < (kPitch + 1023) / 1024; j++) {
            const uint32_t piece = j * 64 + lane;
            if (piece < kPitch / 16 && piece < (ns + 1) / 2 * 16)
              lds_dma16(w, from + min((piece ^ (lr % 16)) * 16, ns * kI8Row - 16), wc + lr * kPitch + j * 1024);
          }
        }
      }
      const auto row_of = [&](uint32_t i) { return x + member[m0 + i] / p.K * stride; };
      if (s0 == 0) {  // the rows' largest
        if (threadIdx.x < kTok) most[threadIdx.x] = 0;
        __syncthreads();
        for (uint32_t i = threadIdx.x; i < nm * steps * 16; i += 256) {
          float v[8];
          load8<kX>(row_of(i / (steps * 16)), i % (steps * 16) * 8, p.H, v);
          uint32_t m = most_of8(v);
          m = max(m, dpp_u32<kDppXor1>(m));
          m = max(m, dpp_u32<kDppXor2>(m));
          m = max(m, dpp_u32<kDppHalfMirror>(m));
          m = max(m, dpp_u32<kDppMirror>(m));
          if (lane % 16 == 0) atomicMax(most + i / (steps * 16), m);
        }
        __syncthreads();
      }
      for (uint32_t i = threadIdx.x; i < nm * ns * 16; i += 256) {
        const uint32_t xr = i / (ns * 16), gr = i - xr * (ns * 16);
        float v[8];
        load8<kX>(row_of(xr), (s0 * 16 + gr) * 8, p.H, v);
        *(uint2 *)(xc + xr * kXPitch + gr * 8) = i8_codes8(v, i8_scale_of(most[xr]));
      }
      dma_barrier();
      const uint32_t xr = min(r, nm - 1);
      for (uint32_t k = wave; k < 2 * ns; k += 4) {
        const mx_i4 b = *(const mx_i4 *)(xc + xr * kXPitch + k * 64 + q * 16);
#pragma unroll
        for (uint32_t i = 0; i < 2; i++)
          acc[i] = i8_mfma16(*(const mx_i4 *)(wc + (16 * i + r) * kPitch + ((4 * k + q) ^ r) * 16), b, acc[i]);
      }
    }
    if (r < kTok)
#pragma unroll
      for (uint32_t i = 0; i < 2; i++)
#pragma unroll
        for (uint32_t j = 0; j < 4; j++) sums[wave][16 * i + 4 * q + j][r] = acc[i][j];
    __syncthreads();
    const uint32_t col = threadIdx.x % 16, t = threadIdx.x / 16;
    if (t < nm && f0 + col < p.F) {
      int gv = 0, uv = 0;
#pragma unroll
      for (uint32_t v = 0; v < 4; v++) gv += sums[v][col][t], uv += sums[v][16 + col][t];
      const float s = i8_scale_of(most[t]);
      h[(uint64_t)member[m0 + t] * pitch + f0 + col] =
          expert_swiglu(i8_value(gv, s, p.gs[row + col]), i8_value(uv, s, p.us[row + col]), p.limit);
    }
    __syncthreads();  // (sums and most)
  }
}

// A work-group: 16 rows of down for all assignments, and y's 16 columns. It quantises the assignments' rows of h; a wave takes
// every eighth of the experts that are used (its assignments 16 at a time), 256 bytes of 16 rows a load, two loads of its own on
// their way.
constexpr uint32_t kFewHq = 56 * 1024;  // the assignments' rows of h in LDS

template <uint32_t kType>
__global__ void __launch_bounds__(512) i8_down_few(I8Experts p, const float *h, uint32_t hpitch, const int32_t *ids, const float *w,
                                                   uint32_t ntok, typename Elem<kType>::T *y, uint64_t stride) {
  struct Slot {
    alignas(16) uint8_t c[16 * 256];  // 16 rows, their 16-byte pieces exchanged by the row
  };
  __shared__ Slot slot0[8];
  __shared__ Slot slot1[8];
  __shared__ __align__(16) uint8_t hq[kFewHq];
  __shared__ __align__(16) int o[kFew * 16];
  __shared__ uint32_t first[512], most[kFew];
  __shared__ uint16_t id[kFew], used[kFew], member[8][kFew];
  __shared__ uint32_t counts[8];
  const uint32_t lane = threadIdx.x & 63, wave = mx_wave(), q = lane / 16, r = lane % 16, A = ntok * p.K;
  const uint32_t pitch = i8_pitch(p.F), r0 = blockIdx.x * 16, lpitch = pitch + 16;
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
  const uint32_t chunks = (pitch + 255) / 256, units = wave < n ? ((n - 1 - wave) / 8 + 1) * chunks : 0;
  const auto load = [&](Slot &s, uint32_t unit) {
    const uint32_t ex = (uint32_t)__builtin_amdgcn_readfirstlane(id[used[wave + unit / chunks * 8]]), k = unit % chunks * 256;
    const uint64_t row = (uint64_t)ex * p.H + r0, rest = (uint64_t)p.E * p.H - row;
    const __amdgpu_buffer_rsrc_t c = mx_buffer((const uint8_t *)p.dc + row * pitch, rest * pitch);
#pragma unroll
    for (uint32_t j = 0; j < 4; j++) {
      const uint32_t lr = 4 * j + lane / 16;
      lds_dma16(c, lr * pitch + k + min(((lane % 16) ^ lr) * 16, min(pitch - k, 256u) - 16), s.c + j * 1024);
    }
  };
  if (units > 0) load(slot0[wave], 0);
  if (units > 1) load(slot1[wave], 1);
  // (Rows of assignments without an expert hold whatever the buffer held: codes that nobody reads.)
  quantize_rows<QT_F32, kFewHq / 8 / 512>(A, pitch, p.F, [&](uint32_t i) { return h + (uint64_t)i * hpitch; }, hq, lpitch, most);
  uint32_t nm = 0;
  const auto use = [&](const Slot &s, uint32_t unit, bool more) {
    // This unit's load has arrived; the next one's four may be outstanding.
    asm volatile("" ::: "memory");
    if (more)
      __builtin_amdgcn_s_waitcnt(0x0f74);
    else
      __builtin_amdgcn_s_waitcnt(0x0f70);
    asm volatile("" ::: "memory");
    const uint32_t k = unit % chunks * 4, ns = min(pitch / 64 - k, 4u);
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
#pragma unroll
    for (uint32_t j = 0; j < 4; j++) a[j] = *(const mx_i4 *)(s.c + r * 256 + ((4 * j + q) ^ r) * 16);
    for (uint32_t m0 = 0; m0 < nm; m0 += 16) {
      const uint32_t as = member[wave][min(m0 + r, nm - 1)];
      mx_i4 c = {0, 0, 0, 0};
      int4 *to = (int4 *)(o + as * 16 + 4 * q);
      if (k != 0) {
        const int4 v = *to;
        c = mx_i4{v.x, v.y, v.z, v.w};
      }
#pragma unroll
      for (uint32_t j = 0; j < 4; j++) {
        if (j >= ns) break;
        c = i8_mfma16(a[j], *(const mx_i4 *)(hq + as * lpitch + (k + j) * 64 + q * 16), c);
      }
      if (m0 + r < nm) *to = make_int4(c[0], c[1], c[2], c[3]);
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
    if (r0 + c >= p.H) continue;
    float s = 0.0f;
    for (uint32_t k = 0; k < p.K; k++) {
      const uint32_t a = t * p.K + k, ex = id[a];
      if (ex < p.E)
        s = __builtin_fmaf(w[a], i8_value(o[a * 16 + c], i8_scale_of(most[a]), p.ds[(uint64_t)ex * p.H + r0 + c]), s);
    }
    y[(uint64_t)t * stride + r0 + c] = (typename Elem<kType>::T)s;
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

// How a call runs. Few assignments, whose rows of h fit LDS, without sorting them.
constexpr uint64_t kChunkBytes = 256 << 20;

struct Plan {
  uint32_t A, rows, hpitch, pitch, chunk, max_tiles;
  bool few;
  uint64_t xc, xs, h, hc, hs, o, sort, order, places, offsets, tiles, n_tiles, bytes;  // the work buffer's parts

  Plan(const moe_i8_experts &e, uint32_t T) {
    A = T * e.n_used;
    few = A <= (e.n_expert <= 32 ? kFew : 96) && A * (i8_pitch(e.n_ff) + 16) <= kFewHq;
    // Tiles of 32, 64 or 128 positions: the more an expert has on average, the fewer times its weights are read.
    const uint32_t mean = A / e.n_expert;
    rows = mean < 24 ? 32 : mean < 96 ? 64 : 128;
    hpitch = (e.n_ff + 3) / 4 * 4;
    pitch = (e.n_embd + 255) / 256 * 256;
    // The values of all assignments at once, or of as many columns at a time as 256 MB hold, about the last-level cache.
    chunk = few ? pitch : std::min<uint64_t>(pitch, std::max<uint64_t>(256, kChunkBytes / (4ull * A) / 256 * 256));
    max_tiles = std::min(A, e.n_expert + A / rows);
    uint64_t at = 0;
    const auto part = [&](uint64_t n) {
      const uint64_t was = at;
      at += (n + 255) / 256 * 256;
      return was;
    };
    h = part((uint64_t)A * hpitch * 4);
    if (!few) {
      xc = part(i8_bytes(T, e.n_embd)), xs = part((uint64_t)T * 4);
      hc = part(i8_bytes(A, e.n_ff)), hs = part((uint64_t)A * 4);
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
    if (at.few) {
      op_by_type(e->x_type, [&](auto t) {
        constexpr uint32_t kX = decltype(t)::value;
        const auto run = [&](auto kernel) {
          op_launch(kernel, (uint64_t)A * ((F + 15) / 16), 256, stream, p, (const typename Elem<kX>::T *)x, x_stride, ids, A, h,
                    at.hpitch);
        };
        if (i8_steps(H) <= 16)
          run(i8_gate_up_few<kX, 16>);
        else
          run(i8_gate_up_few<kX, 20>);
      });
      op_by_type(e->y_type, [&](auto t) {
        constexpr uint32_t kY = decltype(t)::value;
        op_launch(i8_down_few<kY>, (H + 15) / 16, 512, stream, p, (const float *)h, at.hpitch, ids, w, ntok, (typename Elem<kY>::T *)y,
                  y_stride);
      });
      return;
    }
    int32_t *order = (int32_t *)(b + at.order), *places = (int32_t *)(b + at.places);
    uint32_t *offsets = (uint32_t *)(b + at.offsets), *nt = (uint32_t *)(b + at.n_tiles);
    MoeTile *tiles = (MoeTile *)(b + at.tiles);
    float *o = (float *)(b + at.o);
    const moe_i8_matrix xq{(int8_t *)(b + at.xc), (float *)(b + at.xs), ntok, H}, hq{(int8_t *)(b + at.hc), (float *)(b + at.hs), A, F};
    sort_launch(ids, A, E, SortOut{order, places, offsets, tiles, nt, at.rows}, b + at.sort, stream);
    i8_quantize_launch(e->x_type, x, x_stride, xq, nullptr, stream);
    const auto run = [&](auto gate_up, auto down, uint32_t bn) {
      const uint64_t cols = bn / 2, parts = (F + cols - 1) / cols;
      op_launch(gate_up, item_blocks(at.max_tiles * parts, parts), 256, stream, p, (const int8_t *)xq.codes, (const float *)xq.scales,
                ntok, (const int32_t *)order, (const MoeTile *)tiles, (const uint32_t *)nt, h, at.hpitch);
      i8_quantize_launch(QT_F32, h, at.hpitch, hq, offsets + E, stream);
      for (uint32_t c = 0; c < at.pitch; c += at.chunk) {
        const uint32_t n = std::min(at.chunk, at.pitch - c);
        op_launch(down, item_blocks((uint64_t)at.max_tiles * (n / bn), n / bn), 256, stream, p, (const int8_t *)hq.codes,
                  (const float *)hq.scales, (const MoeTile *)tiles, (const uint32_t *)nt, c, n, o);
        combine_launch(QT_F32, o, n, ntok, K, std::min(n, H - c), places, w, e->y_type, (uint8_t *)y + (uint64_t)c * op_size(e->y_type),
                       y_stride, stream);
      }
    };
    if (at.rows == 32) run(i8_gate_up_tiles<1, 1>, i8_down_tiles<1, 1>, 256);
    if (at.rows == 64) run(i8_gate_up_tiles<1, 2>, i8_down_tiles<1, 2>, 128);
    if (at.rows == 128) run(i8_gate_up_tiles<2, 2>, i8_down_tiles<2, 2>, 128);
  });
}

}  // extern "C"
