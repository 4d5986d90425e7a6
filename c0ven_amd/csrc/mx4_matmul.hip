// The products of MX4 matrices (moe_mx4_matmul_async, moe_mx4_linear_async).
#include "mx4.h"
#include "mx4_api.h"
#include "mx4_gemm.h"
#include "ops.h"

#include <algorithm>
#include <type_traits>

namespace c0ven {

// Few rows of x (at most 16): y = x w^T is bound by reading w, and by its loads: 16 rows' 64 bytes are a clock a lane. So a
// row's scales come for four steps of 128 at a time (one by one: as long as the codes; 16 x 8192 x 8192 22.7 us, now 18.9).
// A work-group has 16 rows of w, its kWaves waves each a run of their k, four steps in use and four more on their way; the
// waves' sums are added in their order. kX kQuantised: x is quantised already (xc, xs); else x are floats of that type
// (QT_F32 is 0), which the work-group quantises into LDS while its first loads of w are on their way (1 x 8192 x 2048 4.7 us,
// 7.6 with a launch for it). 1 x 16384 x 8192: 20 us, 3.5 TB/s.
constexpr uint32_t kQuantised = ~0u;
constexpr uint32_t kFewRows = 16;    // (16 x 4096 x 4096 7.5 us, 17 rows by tiles 11.9; 8192 x 8192 18.0 and 18.3)
constexpr uint32_t kFewLds = 16384;  // the most values of x that a work-group quantises for itself

template <uint32_t kX, uint32_t kType, int kWaves>
__global__ void __launch_bounds__(64 * kWaves)
    mx4_few(const void *x, uint64_t x_stride, const uint8_t *xc, const uint8_t *xs, const uint8_t *wc, const uint8_t *ws,
            uint32_t M, uint32_t N, uint32_t cols, typename Elem<kType>::T *y, uint64_t stride) {
  constexpr bool kFloats = kX != kQuantised;
  constexpr uint32_t kCodes = kFloats ? kFewLds / 2 + 16 * kFewRows : 16;
  __shared__ __align__(16) uint8_t lc[kCodes];
  __shared__ __align__(16) uint8_t ls[kFloats ? kFewLds / 32 : 16];
  __shared__ float sums[kWaves][16][17];
  const uint32_t lane = threadIdx.x & 63, wave = mx_wave(), q = lane / 16, r = lane % 16, steps = mx_steps(cols);
  const uint32_t n0 = blockIdx.x * 16, per = (steps + kWaves - 1) / kWaves;
  const uint32_t k0 = min(wave * per, steps), k1 = min(k0 + per, steps);
  const uint64_t row = (uint64_t)min(n0 + r, N - 1) * steps;
  const uint32_t m = min(r, M - 1);
  constexpr int kAhead = 4;
  struct Ahead {
    mx_i4 a[kAhead], b[kAhead];
    uint32_t sa[kAhead], sb[kAhead];
  } one, two;
  const auto words = [&](uint32_t (&to)[kAhead], const uint8_t *from, uint32_t k) {  // a row's scales from step k on
    if (k + kAhead <= steps) {
      struct __attribute__((packed, aligned(4))) Words {
        uint32_t w[kAhead];
      };
      const Words v = *(const Words *)(from + k * 4);
#pragma unroll
      for (int j = 0; j < kAhead; j++) to[j] = v.w[j];
    } else {
#pragma unroll
      for (int j = 0; j < kAhead; j++)
        if (k + j < k1) to[j] = *(const uint32_t *)(from + (k + j) * 4);
    }
  };
  const auto load = [&](Ahead &to, uint32_t k) {
#pragma unroll
    for (int j = 0; j < kAhead; j++) {
      if (k + j >= k1) break;
      to.a[j] = *(const mx_i4 *)(wc + (row + k + j) * 64 + q * 16);
      if constexpr (!kFloats) to.b[j] = *(const mx_i4 *)(xc + ((uint64_t)m * steps + k + j) * 64 + q * 16);
    }
    words(to.sa, ws + row * 4, k);
    if constexpr (!kFloats) words(to.sb, xs + (uint64_t)m * steps * 4, k);
  };
  load(one, k0);
  const uint32_t pitch = steps * 64 + 16;
  if constexpr (kFloats) {
    typedef typename Elem<kX>::T X;
    for (uint32_t i = threadIdx.x; i < M * steps * 16; i += 64 * kWaves) {
      const uint32_t xr = i / (steps * 16), g = i - xr * (steps * 16);
      const X *from = (const X *)x + xr * x_stride;
      float v[8];
      load8<kX>(from, g * 8, cols, v);
      uint32_t s;
      *(uint32_t *)(lc + xr * pitch + g * 4) = mx_quantize8(v, s);
      if (g % 4 == 0) ls[xr * steps * 4 + g / 4] = (uint8_t)s;
    }
    __syncthreads();
  }
  mx_f4 c = {0, 0, 0, 0};
  const auto use = [&](Ahead &v, uint32_t k) {
#pragma unroll
    for (int j = 0; j < kAhead; j++) {
      if (k + j >= k1) break;
      if constexpr (kFloats) {
        v.b[j] = *(const mx_i4 *)(lc + m * pitch + (k + j) * 64 + q * 16);
        v.sb[j] = *(const uint32_t *)(ls + (m * steps + k + j) * 4);
      }
      c = mx_mfma16<0, 0>(v.a[j], v.b[j], c, v.sa[j] >> (8 * q), v.sb[j] >> (8 * q));
    }
  };
  for (uint32_t k = k0; k < k1; k += 2 * kAhead) {
    if (k + kAhead < k1) load(two, k + kAhead);
    use(one, k);
    if (k + 2 * kAhead < k1) load(one, k + 2 * kAhead);
    use(two, k + kAhead);
  }
#pragma unroll
  for (int i = 0; i < 4; i++) sums[wave][r][4 * q + i] = c[i];
  __syncthreads();
  for (uint32_t i = threadIdx.x; i < M * 16; i += 64 * kWaves) {
    float s = 0.0f;
#pragma unroll
    for (int v = 0; v < kWaves; v++) s += sums[v][i / 16][i % 16];
    if (n0 + i % 16 < N) y[(uint64_t)(i / 16) * stride + n0 + i % 16] = (typename Elem<kType>::T)s;
  }
}

// The sums of `parts` parts of y, each M x N, in their order.
template <uint32_t kType>
__global__ void __launch_bounds__(256) mx4_join(const float *sums, uint32_t parts, uint32_t M, uint32_t N,
                                                typename Elem<kType>::T *y, uint64_t stride) {
  const uint64_t n = (uint64_t)M * N, i = (uint64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= n) return;
  float s = 0.0f;
  for (uint32_t p = 0; p < parts; p++) s += sums[p * n + i];
  y[i / N * stride + i % N] = (typename Elem<kType>::T)s;
}

// A tile of y a work-group, k split into parts of `span` stages (256 each); part p's sums go to y + p * part. Work-groups to
// tiles so that an XCD has neighbours: eight tiles down, then across. The 256 tile takes eight waves, two a SIMD (four with
// 256 sums a lane: 177 us at 4096 x 8192 x 8448, 166 with eight). 4096 x 8192 x 8192, after x's quantisation: 166 us on
// average, 3.3 PFLOP/s (145 at least); called back to back 181, x 8448 (rows that are not a power of two apart) 170. Of these
// 137 and 132 remained in a copy without the loop's loads: what the loads add is the wait for a stage that 64 KB a CU cannot hide, since two stages fill LDS.
template <uint32_t kType, int TM, int TN, int kWaves>
__global__ void __launch_bounds__(64 * kWaves, 2)
    mx4_gemm(const uint8_t *xc, const uint8_t *xs, const uint8_t *wc, const uint8_t *ws, uint32_t M, uint32_t N,
             uint32_t steps, uint32_t span, typename Elem<kType>::T *y, uint64_t stride, uint64_t part) {
  typedef MxTile<TM, TN, 2, false, false, kWaves> Tile;
  constexpr int BM = Tile::BM, BN = Tile::BN;
  typedef typename Elem<kType>::T T;
  __shared__ typename Tile::Stage s0;
  __shared__ typename Tile::Stage s1;
  __shared__ typename Tile::Scales scales;
  const uint32_t tm = (M + BM - 1) / BM, tn = (N + BN - 1) / BN, stages = (steps + 1) / 2;
  const uint32_t parts = (stages + span - 1) / span, all = tm * tn * parts;
  const uint32_t per = (all + 7) / 8, id = blockIdx.x % 8 * per + blockIdx.x / 8;
  if (blockIdx.x / 8 >= per || id >= all) return;
  const uint32_t p = id / (tm * tn), t = id % (tm * tn), group = t / (8 * tn), rows = min(tm - group * 8, 8u);
  const uint32_t m0 = (group * 8 + t % (8 * tn) % rows) * BM, n0 = t % (8 * tn) / rows * BN;
  const uint32_t k0 = p * span, k1 = min(k0 + span, stages);
  const auto same = [](uint32_t r) { return r; };
  const MxSource<BM, kWaves> sx(xc + (uint64_t)m0 * steps * 64, xs + (uint64_t)m0 * steps * 4, M - m0, steps, same);
  const MxSource<BN, kWaves> sw(wc + (uint64_t)n0 * steps * 64, ws + (uint64_t)n0 * steps * 4, N - n0, steps, same);
  Tile c;
  c.run(
      s0, s1, scales, k1 - k0,
      [&](typename Tile::Stage &s, uint32_t k) { sx.load(k0 + k, s.x), sw.load(k0 + k, s.w); },
      [&](typename Tile::Scales &s, uint32_t k) { sx.load_scales(k0 + k, s.x), sw.load_scales(k0 + k, s.w); });
  __builtin_amdgcn_s_barrier();  // (the stages' LDS is used again)
  // Each wave's 32 rows at a time through its part of LDS, so that a row's neighbours are stored together.
  const uint32_t lane = threadIdx.x & 63, wave = mx_wave(), q = lane / 32, r = lane % 32;
  constexpr uint32_t kWide = 32 * TN, kPitch = kWide + 4;
  constexpr uint32_t kHalf = kWaves / 2;
  float *mine = (float *)(wave < kHalf ? (uint8_t *)&s0 : (uint8_t *)&s1) + wave % kHalf * 32 * kPitch;
  static_assert(kHalf * 32 * kPitch * 4 <= sizeof(s0), "half the waves' rows in a stage");
  const uint32_t wm = m0 + Tile::x_row(), wn = n0 + Tile::w_row();
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

// How a product of M rows with N rows runs: tiles of 64 t by 64 t, k in parts of span stages of 256. The largest tile that
// still gives most CUs one (a 256 tile moves a quarter of the bytes of a 64 tile through LDS per product): 2048 x 8192 x 4096
// with 256 tiles (256 of them) 51 us, 128 58, 64 82; 1024 x 8192 x 8192 with 256 tiles (128) 72, 128 (512) 56, 64 80; 512 x
// 8192 x 8192 with 128 (256) 40, 64 44. If even the smallest leaves CUs without one, the k axis is split: 64 x 4096 x 8192
// 17.6 us (in one 23.5), 17 x 1024 x 8192 13 (22).
struct Plan {
  uint32_t tile = 1, span, parts = 1;
  uint64_t tiles;
  Plan(uint32_t M, uint32_t N, uint32_t steps) {
    const auto count = [&](uint64_t t) { return ((M + 64 * t - 1) / (64 * t)) * ((N + 64 * t - 1) / (64 * t)); };
    for (uint32_t t : {4u, 2u})
      if (count(t) >= 200) {
        tile = t;
        break;
      }
    tiles = count(tile);
    const uint32_t stages = (steps + 1) / 2;
    span = stages;
    if (tile == 1 && tiles < 200) {
      const uint32_t want = (uint32_t)std::min<uint64_t>(400 / tiles, stages / 2);
      if (want > 1) span = (stages + want - 1) / want;
    }
    parts = (stages + span - 1) / span;
  }
  uint64_t bytes(uint32_t M, uint32_t N) const { return parts > 1 ? (uint64_t)parts * M * N * 4 : 0; }
};

template <uint32_t kX>
void launch_few(const void *x, uint64_t x_stride, const uint8_t *xc, const uint8_t *xs, uint32_t M, const moe_mx4_matrix *w,
                uint32_t y_type, void *y, uint64_t stride, void *stream) {
  const uint32_t N = w->rows, blocks = (N + 15) / 16;
  op_by_type(y_type, [&](auto t) {
    constexpr uint32_t kType = decltype(t)::value;
    const auto run = [&](auto kernel, uint32_t waves) {
      op_launch(kernel, blocks, 64 * waves, stream, x, x_stride, xc, xs, (const uint8_t *)w->codes,
                (const uint8_t *)w->scales, M, N, w->cols, (typename Elem<kType>::T *)y, stride);
    };
    // Sixteen waves a work-group where there are few of them, for a long k (16 x 2048 x 8192 10.1 us, with four 11.1; x 2048
    // 7.0 and 6.6) and for many values to quantise (4 x 512 x 1024 3.2 us, with four 3.6; 16 x 2048 x 1024 3.9 and 5.6; 1 x
    // 2048 x 1024 3.2 and 2.9). With more work-groups four hide each other's latency (4 x 16384 x 2048 8.4 us, 16: 10.0).
    const bool many = kX == kQuantised ? mx_steps(w->cols) >= 64 : M * mx_steps(w->cols) * kMxRow >= 4096;
    if (blocks <= 512 && many)
      run(mx4_few<kX, kType, 16>, 16);
    else
      run(mx4_few<kX, kType, 4>, 4);
  });
}

void launch_matmul(const uint8_t *xc, const uint8_t *xs, uint32_t M, const moe_mx4_matrix *w, uint32_t y_type, void *y,
                   uint64_t stride, void *work, void *stream) {
  const uint32_t N = w->rows, steps = mx_steps(w->cols);
  if (M <= kFewRows) return launch_few<kQuantised>(nullptr, 0, xc, xs, M, w, y_type, y, stride, stream);
  const Plan p(M, N, steps);
  const auto tiles = [&](auto t, void *to, uint64_t to_stride) {
    constexpr uint32_t kType = decltype(t)::value;
    const auto run = [&](auto kernel, uint32_t waves) {
      op_launch(kernel, (p.tiles * p.parts + 7) / 8 * 8, 64 * waves, stream, xc, xs, (const uint8_t *)w->codes,
                (const uint8_t *)w->scales, M, N, steps, p.span, (typename Elem<kType>::T *)to, to_stride,
                (uint64_t)M * N);
    };
    if (p.tile == 4) run(mx4_gemm<kType, 4, 2, 8>, 8);
    if (p.tile == 2) run(mx4_gemm<kType, 2, 2, 4>, 4);
    if (p.tile == 1) run(mx4_gemm<kType, 1, 1, 4>, 4);
  };
  if (p.parts == 1) return op_by_type(y_type, [&](auto t) { tiles(t, y, stride); });
  tiles(std::integral_constant<uint32_t, QT_F32>(), work, N);
  op_by_type(y_type, [&](auto t) {
    constexpr uint32_t kType = decltype(t)::value;
    op_launch(mx4_join<kType>, ((uint64_t)M * N + 255) / 256, 256, stream, (const float *)work, p.parts, M, N,
              (typename Elem<kType>::T *)y, stride);
  });
}

void op_results(uint64_t M, uint64_t N) { op_require(M * N <= 1ull << 38, "y of more than 2^38 elements"); }

// x's rows quantised, in a work buffer.
uint64_t quantised_bytes(uint32_t rows, uint32_t cols) {
  return moe_mx4_code_bytes(rows, cols) + (moe_mx4_scale_bytes(rows, cols) + 15) / 16 * 16;
}
// The rows that the few-rows kernel quantises for itself: another launch costs more than M cols / 2048 rounds of it.
bool quantises_itself(uint32_t M, uint32_t cols) {
  return M <= kFewRows && (uint64_t)M * mx_steps(cols) * kMxRow <= kFewLds;
}

}  // namespace

extern "C" {

MOE_API uint64_t moe_mx4_matmul_work_bytes(const moe_mx4_matrix *w, uint32_t ntok) {
  if (!w || !mx4_sizes(*w) || ntok <= kFewRows || ntok > kMxMostRows || !w->rows) return 0;
  return Plan(ntok, w->rows, mx_steps(w->cols)).bytes(ntok, w->rows);
}

MOE_API moe_status moe_mx4_matmul_async(int32_t device, const moe_mx4_matrix *x, const moe_mx4_matrix *w,
                                        uint32_t y_type, void *y, uint64_t y_stride, void *work, uint64_t work_bytes,
                                        void *stream) {
  return op_guarded([&] {
    op_mx4(x);
    op_mx4(w);
    op_require(x->cols == w->cols, "x and w must have the same cols");
    op_results(x->rows, w->rows);
    op_rows(y, y_stride, w->rows ? x->rows : 0, w->rows, y_type);
    op_work(work, work_bytes, moe_mx4_matmul_work_bytes(w, x->rows));
    if (!x->rows || !w->rows) return;
    OnDevice on(device);
    launch_matmul(x->codes, x->scales, x->rows, w, y_type, y, y_stride, work, stream);
  });
}

MOE_API uint64_t moe_mx4_linear_work_bytes(const moe_mx4_matrix *w, uint32_t ntok) {
  if (!w || !mx4_sizes(*w) || ntok > kMxMostRows || quantises_itself(ntok, w->cols)) return 0;
  return quantised_bytes(ntok, w->cols) + moe_mx4_matmul_work_bytes(w, ntok);
}

MOE_API moe_status moe_mx4_linear_async(int32_t device, uint32_t x_type, const void *x, uint64_t x_stride,
                                        uint32_t ntok, const moe_mx4_matrix *w, uint32_t y_type, void *y,
                                        uint64_t y_stride, void *work, uint64_t work_bytes, void *stream) {
  return op_guarded([&] {
    op_mx4(w);
    op_rows(x, x_stride, ntok, w->cols, x_type);
    op_rows(y, y_stride, w->rows ? ntok : 0, w->rows, y_type);
    op_require(ntok <= kMxMostRows, "at most 2^27 tokens");
    op_results(ntok, w->rows);
    op_work(work, work_bytes, moe_mx4_linear_work_bytes(w, ntok));
    if (!ntok || !w->rows) return;
    OnDevice on(device);
    if (quantises_itself(ntok, w->cols))
      return op_by_type(x_type, [&](auto t) {
        launch_few<decltype(t)::value>(x, x_stride, nullptr, nullptr, ntok, w, y_type, y, y_stride, stream);
      });
    uint8_t *xc = (uint8_t *)work, *xs = xc + moe_mx4_code_bytes(ntok, w->cols);
    const moe_mx4_matrix xm{xc, xs, ntok, w->cols};
    mx4_quantize_launch(x_type, x, x_stride, xm, stream);
    launch_matmul(xc, xs, ntok, w, y_type, y, y_stride, (uint8_t *)work + quantised_bytes(ntok, w->cols), stream);
  });
}

}  // extern "C"
