// The products of I8 matrices (moe_i8_matmul_async, moe_i8_linear_async). The sums are exact in 32 bits (65536 products of at most
// 2^14), so that neither tiles nor a split k change a result.
#include "i8_api.h"
#include "i8_few.h"
#include "i8_gemm.h"

#include <algorithm>
#include <type_traits>

namespace c0ven {

// Few rows of x (at most 16): y = x w^T is bound by reading w. A work-group has 16 rows of w, its kWaves waves each a run of their
// k, four steps of 64 in use and four more on their way; the waves' sums are added in LDS. kX kQuantised: x is quantised already
// (xc, xs); else x are floats of that type, which the work-group quantises into LDS while its first loads of w are on their way.
constexpr uint32_t kQuantised = ~0u;
constexpr uint32_t kFewRows = 16;
constexpr uint32_t kFewLds = 16384;  // the most values of x that a work-group quantises for itself

template <uint32_t kX, uint32_t kType, int kWaves>
__global__ void __launch_bounds__(64 * kWaves)
    i8_few(const void *x, uint64_t x_stride, const int8_t *xc, const float *xs, const int8_t *wc, const float *ws, uint32_t M,
           uint32_t N, uint32_t cols, typename Elem<kType>::T *y, uint64_t stride) {
  constexpr bool kFloats = kX != kQuantised;
  __shared__ __align__(16) uint8_t lc[kFloats ? kFewLds + 16 * kFewRows : 16];
  __shared__ uint32_t ls[kFewRows];
  __shared__ int sums[kWaves][16][17];
  const uint32_t lane = threadIdx.x & 63, wave = mx_wave(), q = lane / 16, r = lane % 16, pitch = i8_pitch(cols);
  const uint32_t steps = pitch / 64, n0 = blockIdx.x * 16, per = (steps / 2 + kWaves - 1) / kWaves * 2;  // (whole lines)
  const uint32_t k0 = min(wave * per, steps), k1 = min(k0 + per, steps), m = min(r, M - 1);
  // Rows of w past the last and steps past the wave's are zeros, so that every load is there and none waits for a branch's.
  const __amdgpu_buffer_rsrc_t w = mx_buffer((const uint8_t *)wc + (uint64_t)n0 * pitch, (uint64_t)(N - n0) * pitch);
  constexpr int kAhead = kWaves == 16 ? 2 : 4;
  struct Ahead {
    mx_i4 a[kAhead], b[kAhead];
  } one, two;
  const auto load = [&](Ahead &to, uint32_t k) {
#pragma unroll
    for (int j = 0; j < kAhead; j++) {
      to.a[j] = __builtin_bit_cast(mx_i4, __builtin_amdgcn_raw_buffer_load_b128(w, k + j < k1 ? r * pitch + q * 16 + (k + j) * 64 : kNowhere, 0, 0));
      if constexpr (!kFloats) to.b[j] = *(const mx_i4 *)(xc + (uint64_t)m * pitch + min(k + j, steps - 1) * 64 + q * 16);
    }
  };
  load(one, k0);
  load(two, k0 + kAhead);
  static_assert(kFewRows * 16 <= 64 * kWaves, "a value of y a thread");
  const uint32_t col = threadIdx.x % 16, row = threadIdx.x / 16;
  const float sw = ws[min(n0 + col, N - 1)];
  float sx = 0.0f;
  if constexpr (kFloats) {
    typedef typename Elem<kX>::T X;
    quantize_rows<kX, kWaves == 16 ? 2 : 4>(M, pitch, cols, [&](uint32_t i) { return (const X *)x + i * x_stride; },
                      [&](uint32_t i, uint32_t c) { return lc + i * (pitch + 16) + c; }, ls);
  } else {
    sx = xs[min(row, M - 1)];
  }
  mx_i4 c = {0, 0, 0, 0};
  const auto use = [&](Ahead &v, uint32_t k) {
#pragma unroll
    for (int j = 0; j < kAhead; j++) {
      if constexpr (kFloats) v.b[j] = *(const mx_i4 *)(lc + m * (pitch + 16) + min(k + j, steps - 1) * 64 + q * 16);
      c = i8_mfma16(v.a[j], v.b[j], c);
    }
  };
#pragma unroll 1
  for (uint32_t k = k0; k < k1; k += 2 * kAhead) {
    use(one, k);
    load(one, k + 2 * kAhead);
    use(two, k + kAhead);
    load(two, k + 3 * kAhead);
  }
#pragma unroll
  for (int i = 0; i < 4; i++) sums[wave][r][4 * q + i] = c[i];
  __syncthreads();
  if (row < M && n0 + col < N) {
    int s = 0;
#pragma unroll
    for (int v = 0; v < kWaves; v++) s += sums[v][row][col];
    if (kFloats) sx = i8_scale_of(ls[row]);
    y[(uint64_t)row * stride + n0 + col] = (typename Elem<kType>::T)i8_value(s, sx, sw);
  }
}

// The sums of `parts` parts, each M x N, and their scales.
template <uint32_t kType>
__global__ void __launch_bounds__(256) i8_join(const int *sums, uint32_t parts, const float *xs, const float *ws, uint32_t M,
                                               uint32_t N, typename Elem<kType>::T *y, uint64_t stride) {
  const uint64_t n = (uint64_t)M * N, i = (uint64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= n) return;
  int s = 0;
  for (uint32_t p = 0; p < parts; p++) s += sums[p * n + i];
  y[i / N * stride + i % N] = (typename Elem<kType>::T)i8_value(s, xs[i / N], ws[i % N]);
}

// A tile of y a work-group, k split into parts of `span` stages; kSums: the sums themselves, part p's to y + p M N, else y's
// values. Work-groups to tiles so that an XCD has neighbours: eight tiles down, then across. The 256 tile has eight waves and
// five buffers. 4096 x 8192 x 8192 on a layer's codes: 247 us, 2.2 POPS, and 254 to 300 with two buffers of each; the clock gives
// way under such codes (on zeros 183 us, 3.0 POPS, and 202 with two buffers), and the matrix instructions alone, on operands
// that stay in registers, take 185 on random ones. Four waves of 128 x 128 each read a third less of LDS but leave a SIMD one wave: 265.
template <uint32_t kType, bool kSums, int TM, int TN, int kWaves>
__global__ void __launch_bounds__(64 * kWaves, 2)
    i8_gemm(const int8_t *xc, const float *xs, const int8_t *wc, const float *ws, uint32_t M, uint32_t N, uint32_t steps,
            uint32_t span, typename Elem<kType>::T *y, uint64_t stride) {
  typedef I8Tile<TM, TN, 2, false, false, kWaves> Tile;
  constexpr int BM = Tile::BM, BN = Tile::BN;
  constexpr bool kFive = BM == 256;
  typedef typename Elem<kType>::T T;
  static_assert(!kSums || sizeof(T) == 4, "sums are 32 bits");
  __shared__ typename Tile::X x0;
  __shared__ typename Tile::X x1;
  __shared__ typename Tile::W w0;
  __shared__ typename Tile::W w1;
  const uint32_t tm = (M + BM - 1) / BM, tn = (N + BN - 1) / BN;
  const uint32_t parts = (steps + span - 1) / span, all = tm * tn * parts;
  const uint32_t per = (all + 7) / 8, id = blockIdx.x % 8 * per + blockIdx.x / 8;
  if (blockIdx.x / 8 >= per || id >= all) return;
  const uint32_t p = id / (tm * tn), t = id % (tm * tn), group = t / (8 * tn), rows = min(tm - group * 8, 8u);
  const uint32_t m0 = (group * 8 + t % (8 * tn) % rows) * BM, n0 = t % (8 * tn) / rows * BN;
  const uint32_t k0 = p * span, k1 = min(k0 + span, steps);
  const auto same = [](uint32_t r) { return r; };
  const I8Source<BM, kWaves> sx(xc + (uint64_t)m0 * steps * kI8Row, M - m0, steps, same);
  const I8Source<BN, kWaves> sw(wc + (uint64_t)n0 * steps * kI8Row, N - n0, steps, same);
  const auto load_x = [&](typename Tile::X &s, uint32_t k) { sx.load(k0 + k, s.b); };
  const auto load_w = [&](typename Tile::W &s, uint32_t k) { sw.load(k0 + k, s.b); };
  Tile c;
  if constexpr (kFive) {
    __shared__ typename Tile::X x2;
    c.template run5<I8Source<BM, kWaves>::kLoads>(x0, x1, x2, w0, w1, k1 - k0, load_x, load_w);
  } else {
    c.run2(x0, x1, w0, w1, k1 - k0, load_x, load_w);
  }
  __builtin_amdgcn_s_barrier();  // (the stages' LDS is used again)
  // Each wave's 32 rows at a time through its part of LDS, so that a row's neighbours are stored together: a lane has four
  // columns, the same of every row.
  const uint32_t lane = threadIdx.x & 63, wave = mx_wave(), q = lane / 32, r = lane % 32;
  constexpr uint32_t kWide = 32 * TN, kPitch = kWide + 4, kFour = kWaves / 4;
  static_assert(64 % (kWide / 4) == 0, "a lane's columns");
  static_assert(kWaves % 4 == 0 && kFour * 32 * kPitch * 4 <= sizeof(x0) && BM == BN, "a quarter of the waves' rows in a buffer");
  const uint32_t b = wave / kFour;
  int *mine = (int *)(b == 0 ? x0.b : b == 1 ? x1.b : b == 2 ? w0.b : w1.b) + wave % kFour * 32 * kPitch;
  const uint32_t wm = m0 + Tile::x_row(), gn = n0 + Tile::w_row() + lane % (kWide / 4) * 4;
  if (kSums) y += (uint64_t)p * M * N;
  const bool whole = gn + 4 <= N && stride % 4 == 0 && ((uintptr_t)y & (4 * sizeof(T) - 1)) == 0;
  float scale[4];
#pragma unroll
  for (uint32_t j = 0; j < 4; j++) scale[j] = kSums || gn + j >= N ? 0.0f : ws[gn + j];
#pragma unroll
  for (int m = 0; m < TM; m++) {
#pragma unroll
    for (int n = 0; n < TN; n++)
#pragma unroll
      for (int j = 0; j < 4; j++)
        *(int4 *)(mine + r * kPitch + 32 * n + 8 * j + 4 * q) =
            make_int4(c.acc[n][m][4 * j], c.acc[n][m][4 * j + 1], c.acc[n][m][4 * j + 2], c.acc[n][m][4 * j + 3]);
    __builtin_amdgcn_s_waitcnt(0xc07f);
    __builtin_amdgcn_wave_barrier();
#pragma unroll 4
    for (uint32_t row = lane / (kWide / 4); row < 32; row += 64 / (kWide / 4)) {
      const int4 v = *(const int4 *)(mine + row * kPitch + lane % (kWide / 4) * 4);
      const uint32_t gm = wm + 32 * m + row;
      if (gm >= M) continue;
      const int s[4] = {v.x, v.y, v.z, v.w};
      const float f = kSums ? 0.0f : xs[gm];
      T e[4];
#pragma unroll
      for (int j = 0; j < 4; j++) {
        if constexpr (kSums)
          e[j] = (T)__int_as_float(s[j]);
        else
          e[j] = (T)i8_value(s[j], f, scale[j]);
      }
      T *to = y + (uint64_t)gm * stride + gn;
      if (whole) {
        struct alignas(4 * sizeof(T)) Four {
          T e[4];
        };
        *(Four *)to = Four{{e[0], e[1], e[2], e[3]}};
      } else {
        for (uint32_t j = 0; j < 4; j++)
          if (gn + j < N) to[j] = e[j];
      }
    }
    __builtin_amdgcn_s_waitcnt(0xc07f);
    __builtin_amdgcn_wave_barrier();
  }
}

}  // namespace c0ven

using namespace c0ven;

namespace {

// How a product of M rows with N rows runs: tiles of 64 t by 64 t, k in parts of span stages of 128. The largest tile that still
// gives most CUs one; if even the smallest leaves CUs without one, the k axis is split.
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
    span = steps;
    if (tile == 1 && tiles < 200) {
      const uint32_t want = (uint32_t)std::min<uint64_t>(400 / tiles, steps / 4);
      if (want > 1) span = (steps + want - 1) / want;
    }
    parts = (steps + span - 1) / span;
  }
  uint64_t bytes(uint32_t M, uint32_t N) const { return parts > 1 ? (uint64_t)parts * M * N * 4 : 0; }
};

template <uint32_t kX>
void launch_few(const void *x, uint64_t x_stride, const int8_t *xc, const float *xs, uint32_t M, const moe_i8_matrix *w,
                uint32_t y_type, void *y, uint64_t stride, void *stream) {
  const uint32_t N = w->rows, blocks = (N + 15) / 16;
  op_by_type(y_type, [&](auto t) {
    constexpr uint32_t kType = decltype(t)::value;
    const auto run = [&](auto kernel, uint32_t waves) {
      op_launch(kernel, blocks, 64 * waves, stream, x, x_stride, xc, xs, (const int8_t *)w->codes, (const float *)w->scales, M, N,
                w->cols, (typename Elem<kType>::T *)y, stride);
    };
    // Sixteen waves a work-group where there are few of them, for a long k (1 x 512 x 16384 quantised 11.7 us, with four 13.8; x
    // 8192 with 2048 rows 7.9 and 8.1; 16 x 4096 x 4096 7.4 and 6.6) and for many values to quantise (8 x 2048 x 2048 5.5, with
    // four 8.0; 4 x 2048 x 2048 5.0 and 5.3; 1 x 2048 x 2048 4.4 and 4.2). With more work-groups four hide each other's latency
    // (1 x 16384 x 8192 25.6, with sixteen 27.5).
    const bool many = kX == kQuantised ? i8_steps(w->cols) >= 64 : M * i8_pitch(w->cols) >= 8192;
    if (blocks <= 512 && many)
      run(i8_few<kX, kType, 16>, 16);
    else
      run(i8_few<kX, kType, 4>, 4);
  });
}

void launch_matmul(const int8_t *xc, const float *xs, uint32_t M, const moe_i8_matrix *w, uint32_t y_type, void *y,
                   uint64_t stride, void *work, void *stream) {
  const uint32_t N = w->rows, steps = i8_steps(w->cols);
  if (M <= kFewRows) return launch_few<kQuantised>(nullptr, 0, xc, xs, M, w, y_type, y, stride, stream);
  const Plan p(M, N, steps);
  const auto tiles = [&](auto t, auto sums, void *to, uint64_t to_stride) {
    constexpr uint32_t kType = decltype(t)::value;
    constexpr bool kSums = decltype(sums)::value;
    const auto run = [&](auto kernel, uint32_t waves) {
      op_launch(kernel, (p.tiles * p.parts + 7) / 8 * 8, 64 * waves, stream, xc, xs, (const int8_t *)w->codes,
                (const float *)w->scales, M, N, steps, p.span, (typename Elem<kType>::T *)to, to_stride);
    };
    if constexpr (!kSums) {
      if (p.tile == 4) run(i8_gemm<kType, kSums, 4, 2, 8>, 8);
      if (p.tile == 2) run(i8_gemm<kType, kSums, 2, 2, 4>, 4);
    }
    if (p.tile == 1) run(i8_gemm<kType, kSums, 1, 1, 4>, 4);
  };
  if (p.parts == 1) return op_by_type(y_type, [&](auto t) { tiles(t, std::false_type(), y, stride); });
  tiles(std::integral_constant<uint32_t, QT_F32>(), std::true_type(), work, N);
  op_by_type(y_type, [&](auto t) {
    constexpr uint32_t kType = decltype(t)::value;
    op_launch(i8_join<kType>, ((uint64_t)M * N + 255) / 256, 256, stream, (const int *)work, p.parts, xs, (const float *)w->scales, M, N,
              (typename Elem<kType>::T *)y, stride);
  });
}

void op_results(uint64_t M, uint64_t N) { op_require(M * N <= 1ull << 38, "y of more than 2^38 elements"); }

// x's rows quantised, in a work buffer.
uint64_t quantised_bytes(uint32_t rows, uint32_t cols) { return i8_bytes(rows, cols) + ((uint64_t)rows * 4 + 15) / 16 * 16; }
// The rows that the few-rows kernel quantises for itself (it takes eight values at a time).
bool quantises_itself(uint32_t M, uint32_t cols) { return !M || (M <= kFewRows && cols >= 8 && M * i8_pitch(cols) <= kFewLds); }

}  // namespace

extern "C" {

MOE_API uint64_t moe_i8_matmul_work_bytes(const moe_i8_matrix *w, uint32_t ntok) {
  if (!w || !i8_sizes(*w) || ntok <= kFewRows || ntok > kI8MostRows || !w->rows) return 0;
  return Plan(ntok, w->rows, i8_steps(w->cols)).bytes(ntok, w->rows);
}

MOE_API moe_status moe_i8_matmul_async(int32_t device, const moe_i8_matrix *x, const moe_i8_matrix *w, uint32_t y_type, void *y,
                                       uint64_t y_stride, void *work, uint64_t work_bytes, void *stream) {
  return op_guarded([&] {
    op_i8(x);
    op_i8(w);
    op_require(x->cols == w->cols, "x and w must have the same cols");
    op_results(x->rows, w->rows);
    op_rows(y, y_stride, w->rows ? x->rows : 0, w->rows, y_type);
    op_work(work, work_bytes, moe_i8_matmul_work_bytes(w, x->rows));
    if (!x->rows || !w->rows) return;
    OnDevice on(device);
    launch_matmul(x->codes, x->scales, x->rows, w, y_type, y, y_stride, work, stream);
  });
}

MOE_API uint64_t moe_i8_linear_work_bytes(const moe_i8_matrix *w, uint32_t ntok) {
  if (!w || !i8_sizes(*w) || ntok > kI8MostRows || quantises_itself(ntok, w->cols)) return 0;
  return quantised_bytes(ntok, w->cols) + moe_i8_matmul_work_bytes(w, ntok);
}

MOE_API moe_status moe_i8_linear_async(int32_t device, uint32_t x_type, const void *x, uint64_t x_stride, uint32_t ntok,
                                       const moe_i8_matrix *w, uint32_t y_type, void *y, uint64_t y_stride, void *work,
                                       uint64_t work_bytes, void *stream) {
  return op_guarded([&] {
    op_i8(w);
    op_rows(x, x_stride, ntok, w->cols, x_type);
    op_rows(y, y_stride, w->rows ? ntok : 0, w->rows, y_type);
    op_require(ntok <= kI8MostRows, "at most 2^27 tokens");
    op_results(ntok, w->rows);
    op_work(work, work_bytes, moe_i8_linear_work_bytes(w, ntok));
    if (!ntok || !w->rows) return;
    OnDevice on(device);
    if (quantises_itself(ntok, w->cols))
      return op_by_type(x_type, [&](auto t) {
        launch_few<decltype(t)::value>(x, x_stride, nullptr, nullptr, ntok, w, y_type, y, y_stride, stream);
      });
    int8_t *xc = (int8_t *)work;
    float *xs = (float *)(xc + i8_bytes(ntok, w->cols));
    i8_quantize_launch(x_type, x, x_stride, moe_i8_matrix{xc, xs, ntok, w->cols}, nullptr, stream);
    launch_matmul(xc, xs, ntok, w, y_type, y, y_stride, (uint8_t *)work + quantised_bytes(ntok, w->cols), stream);
  });
}

}  // extern "C"
