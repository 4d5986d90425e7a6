// The products of I8 matrices (moe_i8_matmul_async, moe_i8_linear_async). The sums are exact in 32 bits (65536 products of at most
// 2^14), so that neither tiles nor a split k change a result.
#include "i8_api.h"
#include "i8_few.h"
#include "i8_gemm.h"

#include <algorithm>
#include <type_traits>

namespace c0ven {

// Few rows of x (at most 16): y = x w^T is bound by reading w. A work-group has 16 rows of w, its kWaves waves each a run of their
// k, four steps of 64 in use and four more on their way; the waves' sums are added in LDS. 1 x 16384 x 8192 25.6 us (5.2 TB/s),
// 8 x 2048 x 2048 with x's quantisation 5.5. kX kQuantised: x is quantised already
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
      const uint32_t at = k + j < k1 ? r * pitch + q * 16 + (k + j) * 64 : kNowhere;
      to.a[j] = __builtin_bit_cast(mx_i4, __builtin_amdgcn_raw_buffer_load_b128(w, at, 0, 0));
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

// Four elements at whatever address.
template <typename T>
struct __attribute__((packed, aligned(sizeof(T)))) Four {
  T e[4];
};

// The sums of `parts` parts, each M x N (fewer than 2^31), and their scales: four columns a thread.
template <uint32_t kType>
__global__ void __launch_bounds__(256) i8_join(const int *sums, uint32_t parts, const float *xs, const float *ws, uint32_t M,
                                               uint32_t N, typename Elem<kType>::T *y, uint64_t stride) {
  typedef typename Elem<kType>::T T;
  const uint32_t across = (N + 3) / 4, i = blockIdx.x * 256 + threadIdx.x, m = i / across, n0 = i % across * 4;
  if (m >= M) return;
  const uint64_t size = (uint64_t)M * N;
  const int *from = sums + (uint64_t)m * N + n0;
  T *to = y + m * stride + n0;
  const float sx = xs[m];
  if (n0 + 4 <= N) {
    int s[4] = {0, 0, 0, 0};
    const Four<float> sw = *(const Four<float> *)(ws + n0);
#pragma unroll 4
    for (uint32_t p = 0; p < parts; p++) {
      const Four<int> v = *(const Four<int> *)(from + p * size);
#pragma unroll
      for (int j = 0; j < 4; j++) s[j] += v.e[j];
    }
    Four<T> o;
#pragma unroll
    for (int j = 0; j < 4; j++) o.e[j] = (T)i8_value(s[j], sx, sw.e[j]);
    *(Four<T> *)to = o;
  } else {
    for (uint32_t j = 0; n0 + j < N; j++) {
      int s = 0;
      for (uint32_t p = 0; p < parts; p++) s += from[p * size + j];
      to[j] = (T)i8_value(s, sx, ws[n0 + j]);
    }
  }
}

// A tile of y a work-group, k split into parts of `span` stages; kSums: the sums themselves, part p's to y + p M N, else y's
// values. Work-groups to tiles so that an XCD has neighbours: eight tiles down, then across. kBuffers: two of x and two of w,
// four of each, or three of x and two of w (the 256 tile's, which has eight waves).
// 4096 x 8192 x 8192 on a layer's codes: 250 us, 2.2 POPS (traced 290, from 248 to 339; 228 on another card). Bound by power there: the
// clock gives way under such codes (on zeros 184 us, 3.0 POPS), and the matrix instructions alone, on operands that stay in registers,
// take 168 to 182 on random ones. On a card where it took 237 it was 247 before the values went out as below, with two buffers of each
// 254 to 300, and with four waves of 128 x 128, which read a third less of LDS but leave a SIMD one wave, 265. Small products are bound
// by latency and by w (17 x 8192 x 8192 14.5 us, 4.7 TB/s), wide ones of a short k by the values' way out (4096 x 8192 x 1024 47 us).
template <uint32_t kType, bool kSums, int TM, int TN, int kWaves, int kBuffers>
__global__ void __launch_bounds__(64 * kWaves, 2)
    i8_gemm(const int8_t *xc, const float *xs, const int8_t *wc, const float *ws, uint32_t M, uint32_t N, uint32_t steps,
            uint32_t span, typename Elem<kType>::T *y, uint64_t stride) {
  typedef I8Tile<TM, TN, 2, false, false, kWaves> Tile;
  constexpr int BM = Tile::BM, BN = Tile::BN;
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
  const uint32_t lane = threadIdx.x & 63, wave = mx_wave(), q = lane / 32, r = lane % 32;
  constexpr uint32_t kWide = 32 * TN, kPitch = kWide + 4, kFour = kWaves / 4;
  const uint32_t wm = m0 + Tile::x_row(), gn = n0 + Tile::w_row() + lane % (kWide / 4) * 4;
  // The scales: a lane's four columns' and one of each 32 rows' (before any store, which a load would wait for).
  float scale[4], row_scale[TM];
#pragma unroll
  for (uint32_t j = 0; j < 4; j++) scale[j] = kSums ? 0.0f : ws[min(gn + j, N - 1)];
#pragma unroll
  for (int m = 0; m < TM; m++) row_scale[m] = kSums ? 0.0f : xs[min(wm + 32 * m + r, M - 1)];
  Tile c;
  if constexpr (kBuffers == 8) {
    __shared__ typename Tile::X x2;
    __shared__ typename Tile::X x3;
    __shared__ typename Tile::W w2;
    __shared__ typename Tile::W w3;
    const auto within_x = [&](typename Tile::X &s, uint32_t k) { sx.load(k0 + k, s.b, k1); };
    const auto within_w = [&](typename Tile::W &s, uint32_t k) { sw.load(k0 + k, s.b, k1); };
    constexpr int kLoads = I8Source<BM, kWaves>::kLoads + I8Source<BN, kWaves>::kLoads;
    c.template run8<kLoads>(x0, x1, x2, x3, w0, w1, w2, w3, k1 - k0, within_x, within_w);
  } else if constexpr (kBuffers == 5) {
    __shared__ typename Tile::X x2;
    c.template run5<I8Source<BM, kWaves>::kLoads>(x0, x1, x2, w0, w1, k1 - k0, load_x, load_w);
  } else {
    c.run2(x0, x1, w0, w1, k1 - k0, load_x, load_w);
  }
  __builtin_amdgcn_s_barrier();  // (the stages' LDS is used again)
  // Each wave's 32 rows at a time through its part of LDS, so that a row's neighbours are stored together: a lane has four
  // columns, the same of every row; whole tiles without a branch (4096 x 8192 x 128 22 us; 36 with a test and a scale's load a row).
  static_assert(64 % (kWide / 4) == 0, "a lane's columns");
  static_assert(kWaves % 4 == 0 && kFour * 32 * kPitch * 4 <= sizeof(x0) && BM == BN, "a quarter of the waves' rows in a buffer");
  const uint32_t b = wave / kFour;
  int *mine = (int *)(b == 0 ? x0.b : b == 1 ? x1.b : b == 2 ? w0.b : w1.b) + wave % kFour * 32 * kPitch;
  if (kSums) y += (uint64_t)p * M * N;
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
    constexpr uint32_t kRows = 64 / (kWide / 4);  // at a time
    const auto value = [&](uint32_t i) {
      const uint32_t row = lane / (kWide / 4) + kRows * i;
      const int4 v = *(const int4 *)(mine + row * kPitch + lane % (kWide / 4) * 4);
      const float f = kSums ? 0.0f : __shfl(row_scale[m], row);
      if constexpr (kSums)
        return Four<T>{{__int_as_float(v.x), __int_as_float(v.y), __int_as_float(v.z), __int_as_float(v.w)}};
      else
        return Four<T>{{(T)i8_value(v.x, f, scale[0]), (T)i8_value(v.y, f, scale[1]), (T)i8_value(v.z, f, scale[2]),
                        (T)i8_value(v.w, f, scale[3])}};
    };
    T *const to = y + (uint64_t)(wm + 32 * m + lane / (kWide / 4)) * stride + gn;
    if (wm + 32 * m + 32 <= M && n0 + Tile::w_row() + kWide <= N) {
#pragma unroll
      for (uint32_t i = 0; i < 32 / kRows; i++) *(Four<T> *)(to + kRows * i * stride) = value(i);
    } else {
#pragma unroll 1
      for (uint32_t i = 0; i < 32 / kRows; i++) {
        const Four<T> v = value(i);
        if (wm + 32 * m + lane / (kWide / 4) + kRows * i < M) {
          if (gn + 4 <= N)
            *(Four<T> *)(to + kRows * i * stride) = v;
          else
            for (uint32_t j = 0; j < 4; j++)
              if (gn + j < N) to[kRows * i * stride + j] = v.e[j];
        }
      }
    }
    __builtin_amdgcn_s_waitcnt(0xc07f);
    __builtin_amdgcn_wave_barrier();
  }
}

}  // namespace c0ven

using namespace c0ven;

namespace {

// How a product of M rows with N rows runs: tiles of 64 t by 64 t, k in parts of span stages of 128. Up to 512 tiles of 64 (two a
// CU with four buffers each) wait for memory's latency: four buffers (128 x 8192 x 8192 23.8 us, with two 50; 512 x 4096 x 4096
// 17.4 and 20.4), and with few tiles parts of k, by what their sums' way through memory costs: a stage takes 220 ns, a part's sums
// are written and read at 310 to the nanosecond, a launch is 1.5 us (17 x 4096 x 4096 in four parts 7.7 us, in one 10.0, in eight
// 9.3; 128 x 2048 x 2048 7.5, in two 8.0). More are fewer loads in larger tiles, if those still fill the 256 CUs and are not half
// empty to a side: tiles of 256 where their rounds are three quarters full (2048 x 8192 x 8192 120 us, tiles of 128 145; 2500 x
// 5120 x 4096, 200 tiles, 55 and 63; but 2678 x 6333 x 4096, 275 tiles, 106 and 91; 4096 x 6144 x 4096, 384, 110 and 109; 100 x
// 100000 x 4096 131 and 114), else tiles of 128, one to a CU with four buffers (512 x 8192 x 8192 46.5, with two 63.8, tiles of 64
// 66) or two with two (1024 x 8192 x 8192 75, with four 89), else tiles of 64 with two (1500 x 1500 x 512 6.5, with four 8.1,
// tiles of 128 8.7; 40 x 40000 x 1024 11.6, 12.8 and 14.6) or, for a long k, four (17 x 100000 x 4096 87, with two 100, tiles of
// 128 105).
struct Plan {
  uint32_t tile, buffers, span, parts = 1;
  uint64_t tiles;
  Plan(uint32_t M, uint32_t N, uint32_t steps) {
    const auto count = [&](uint64_t t) { return ((M + 64 * t - 1) / (64 * t)) * ((N + 64 * t - 1) / (64 * t)); };
    const uint32_t side = std::min(M, N);
    span = steps;
    if (count(1) <= 512) {
      tile = 1, buffers = 8;
      uint64_t least = ~0ull;
      for (uint32_t p = 1; p <= std::max<uint64_t>(1, std::min<uint64_t>(512 / count(1), steps)); p++) {
        const uint32_t of = (steps + p - 1) / p;
        const uint64_t ns = of * 220ull + (p > 1 ? 1500 + (uint64_t)p * M * N / 310 : 0);
        if (ns < least) least = ns, span = of;
      }
      parts = (steps + span - 1) / span;
    } else if (side > 128 && count(4) * 4 >= (count(4) + 255) / 256 * 256 * 3) {
      tile = 4, buffers = 5;
    } else if (side > 64 && count(2) >= 200) {
      tile = 2, buffers = count(2) <= 256 ? 8 : 4;
    } else {
      tile = 1, buffers = steps >= 24 ? 8 : 4;
    }
    tiles = count(tile);
  }
  uint64_t bytes(uint32_t M, uint32_t N) const { return parts > 1 ? (uint64_t)parts * M * N * 4 : 0; }
};

// Quantised rows that the few-rows kernel takes, else the tiles do. Above eight, on weights of 32 MB and more, every line of w's is
// worth more than a launch, and the tiles have more of them on their way (16 x 8192 x 8192 16.4 us and 19.2,
// 16 x 16384 x 4096 16.3 and 20.4; 8 x 8192 x 8192 15.7 and 16.8, 16 x 4096 x 4096 7.5 and 6.2).
bool few_rows(uint32_t M, const moe_i8_matrix &w) {
  return M <= 8 || (M <= kFewRows && (uint64_t)w.rows * i8_pitch(w.cols) < 32u << 20);
}

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
  if (few_rows(M, *w)) return launch_few<kQuantised>(nullptr, 0, xc, xs, M, w, y_type, y, stride, stream);
  const Plan p(M, N, steps);
  const auto tiles = [&](auto t, auto sums, void *to, uint64_t to_stride) {
    constexpr uint32_t kType = decltype(t)::value;
    constexpr bool kSums = decltype(sums)::value;
    const auto run = [&](auto kernel, uint32_t waves) {
      op_launch(kernel, (p.tiles * p.parts + 7) / 8 * 8, 64 * waves, stream, xc, xs, (const int8_t *)w->codes,
                (const float *)w->scales, M, N, steps, p.span, (typename Elem<kType>::T *)to, to_stride);
    };
    if constexpr (!kSums) {
      if (p.tile == 4) return run(i8_gemm<kType, kSums, 4, 2, 8, 5>, 8);
      if (p.tile == 2) return p.buffers == 8 ? run(i8_gemm<kType, kSums, 2, 2, 4, 8>, 4) : run(i8_gemm<kType, kSums, 2, 2, 4, 4>, 4);
      if (p.buffers == 4) return run(i8_gemm<kType, kSums, 1, 1, 4, 4>, 4);
    }
    run(i8_gemm<kType, kSums, 1, 1, 4, 8>, 4);
  };
  if (p.parts == 1) return op_by_type(y_type, [&](auto t) { tiles(t, std::false_type(), y, stride); });
  tiles(std::integral_constant<uint32_t, QT_F32>(), std::true_type(), work, N);
  op_by_type(y_type, [&](auto t) {
    constexpr uint32_t kType = decltype(t)::value;
    op_launch(i8_join<kType>, ((uint64_t)M * ((N + 3) / 4) + 255) / 256, 256, stream, (const int *)work, p.parts, xs,
              (const float *)w->scales, M, N, (typename Elem<kType>::T *)y, stride);
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
  if (!w || !i8_sizes(*w) || ntok > kI8MostRows || !w->rows || few_rows(ntok, *w)) return 0;
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
