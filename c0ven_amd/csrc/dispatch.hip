// Tokens sorted by expert and back (moe_dispatch_async, moe_combine_async) and the gradients of both.
//
// All of it moves rows: bound by memory. The sort is a stable counting sort of the ids; the rows are read and written 16 bytes
// a lane, a wave a run of 64 such pieces of one token, whose places are then the wave's (scalar loads). 16384 tokens of 10 ranks and
// rows of 4 KB: dispatched in 153 us (15 of them the sort's, the rows at 5.2 TB/s), combined in 123 (5.9, mostly read), the gradients
// of 4096 in 97 (5.5); wide accesses alone read 7.1 TB/s and write 6.8. A few hundred tokens are bound by launches and the sort's
// steps: 999 of 4 ranks and rows of 10 KB 17.9, 100 of 10 ranks 6.1, 8 combined 3.9.
#include "dispatch.h"
#include "experts.h"
#include "mx4_api.h"
#include "sort.h"

#include <algorithm>

namespace c0ven {

// ---- the sort

__global__ void __launch_bounds__(1024) sort_count(const int32_t *ids, uint32_t A, uint32_t E, uint32_t slice, uint32_t *counts) {
  count_slice(ids, A, E, slice, counts);
}
template <bool kOnce>
__global__ void __launch_bounds__(1024) sort_place(const int32_t *ids, uint32_t A, uint32_t E, uint32_t slice, const uint32_t *counts,
                                                   SortOut out) {
  place_slice<kOnce>(ids, A, E, slice, gridDim.x, counts, out);
}

// ---- rows

// kN neighbouring elements: 16 bytes at whatever address, or one element (rows shorter than 16 bytes). Rows pass through once and
// are far more than a cache holds, so they are loaded and stored past it (16384 x 10 rows of 4 KB: dispatched in 153 us, 157
// through the caches; combined in 123, 140; both gradients of 4096 x 10 in 98, 112).
typedef uint32_t Quad __attribute__((ext_vector_type(4), aligned(2)));
template <uint32_t kType, uint32_t kN>
struct Few {
  typedef typename Elem<kType>::T T;
  struct Pack {
    T e[kN];
  };
  typedef typename std::conditional<kN == 1, T, Quad>::type V;
  V v;
  __device__ __forceinline__ void load(const T *p) {
    if constexpr (kN == 1)
      v = *p;
    else
      v = __builtin_nontemporal_load((const Quad *)p);
  }
  __device__ __forceinline__ void store(T *p) const {
    if constexpr (kN == 1)
      *p = v;
    else
      __builtin_nontemporal_store(v, (Quad *)p);
  }
  __device__ __forceinline__ float operator[](uint32_t j) const {
    if constexpr (kN == 1) {
      return (float)v;
    } else {
      return (float)__builtin_bit_cast(Pack, v).e[j];
    }
  }
  static __device__ __forceinline__ Few of(const float f[kN]) {
    Few r;
    Pack p;
#pragma unroll
    for (uint32_t j = 0; j < kN; j++) p.e[j] = (T)f[j];
    if constexpr (kN == 1)
      r.v = p.e[0];
    else
      r.v = __builtin_bit_cast(V, p);
    return r;
  }
};
template <uint32_t kType>
constexpr uint32_t kWhole = 16 / sizeof(typename Elem<kType>::T);  // elements of a whole piece

// Which row (of n) and which of its pieces of kN elements a lane has: kWide: a wave's 64 pieces are one row's, so that what goes by
// the row is scalar; else the lanes follow one another through the rows. The last piece of a row ends with it, and so shares some
// elements with the one before (both write the same).
template <bool kWide, uint32_t kN, typename F>
__device__ __forceinline__ void each_piece(uint32_t n, uint32_t cols, F f) {
  const uint32_t pieces = (cols + kN - 1) / kN;
  if (kWide) {
    const uint32_t runs = (pieces + 63) / 64, wave = blockIdx.x * 4 + (uint32_t)__builtin_amdgcn_readfirstlane(threadIdx.x / 64);
    const uint32_t row = wave / runs, piece = (wave - row * runs) * 64 + threadIdx.x % 64;
    if (row < n && piece < pieces) f(row, min(piece * kN, cols - kN));
  } else {
    const uint32_t i = blockIdx.x * 256 + threadIdx.x, row = i / pieces;
    if (row < n) f(row, min((i - row * pieces) * kN, cols - kN));
  }
}

// A value that is loaded here, whatever branch uses it (the compiler moves scalar loads into the branches, one wait each: a
// dispatch's ten stores waited for ten of them).
template <bool kWide, typename T>
__device__ __forceinline__ void loaded(T &v) {
  if (kWide)
    asm volatile("" : "+s"(v));
  else
    asm volatile("" : "+v"(v));
}

// Each token's row to its ranks' places.
template <bool kWide, uint32_t kType, uint32_t kN>
__global__ void __launch_bounds__(256) dispatch_rows(const typename Elem<kType>::T *__restrict__ x, uint64_t x_stride, uint32_t ntok,
                                                     uint32_t K, uint32_t cols, const int32_t *__restrict__ places,
                                                     typename Elem<kType>::T *__restrict__ xs, uint64_t xs_stride) {
  each_piece<kWide, kN>(ntok, cols, [&](uint32_t t, uint32_t c) {
    Few<kType, kN> v;
    v.load(x + t * x_stride + c);
    int32_t to[16];
#pragma unroll
    for (uint32_t k = 0; k < 16; k++) to[k] = places[t * K + min(k, K - 1)];
#pragma unroll
    for (uint32_t k = 0; k < 16; k++) loaded<kWide>(to[k]);
#pragma unroll
    for (uint32_t k = 0; k < 16; k++) {
      if (k >= K) break;
      if (to[k] >= 0) v.store(xs + (uint64_t)(uint32_t)to[k] * xs_stride + c);
    }
  });
}

// At most kFewIds ids: the sort and the rows in one launch, a work-group every parts-th 256 pieces of a token, whose places its waves
// count themselves (lower ids, and equal ones before), and the last work-group the offsets. cols 0: no rows. 100 tokens of 10 ranks
// 6.0 us, in two launches 9.8; 250 9.3 and 11; 400 12.8 and 12.5: each token's work-group reads all ids.
constexpr uint32_t kFewIds = 2560;
template <uint32_t kType, uint32_t kN>
__global__ void __launch_bounds__(256) dispatch_few(const int32_t *ids, uint32_t ntok, uint32_t K, uint32_t E,
                                                    const typename Elem<kType>::T *x, uint64_t x_stride, uint32_t cols,
                                                    typename Elem<kType>::T *xs, uint64_t xs_stride, uint32_t parts, SortOut out) {
  constexpr uint32_t kKeys = 16, kKey = 4096;  // (ids a lane at a time; above an assignment)
  static_assert(kFewIds <= kKey, "an assignment in a key");
  const uint32_t A = ntok * K, lane = threadIdx.x & 63;
  if (blockIdx.x == gridDim.x - 1) {
    __shared__ uint32_t n[kMostExperts];
    __shared__ uint32_t sums[4];
    for (uint32_t e = threadIdx.x; e < kMostExperts; e += 256) n[e] = 0;
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < A; i += 256)
      if ((uint32_t)ids[i] < E) atomicAdd(n + (uint32_t)ids[i], 1u);
    __syncthreads();
    const uint32_t e = 2 * threadIdx.x, n0 = n[e], n1 = n[e + 1];
    uint32_t place = n0 + n1;
    for (uint32_t d = 1; d < 64; d *= 2) {
      const uint32_t p = (uint32_t)__shfl_up((int)place, d, 64);
      if (lane >= d) place += p;
    }
    if (lane == 63) sums[threadIdx.x / 64] = place;
    __syncthreads();
    uint32_t total = 0;
    for (uint32_t v = 0; v < 4; v++) {
      if (v < threadIdx.x / 64) place += sums[v];
      total += sums[v];
    }
    if (e < E) out.offsets[e] = place - n0 - n1;
    if (e + 1 < E) out.offsets[e + 1] = place - n1;
    if (threadIdx.x == 0) out.offsets[E] = total;
    for (uint32_t i = total + threadIdx.x; i < A; i += 256) out.order[i] = -1;
    return;
  }
  __shared__ uint32_t places[16];
  const uint32_t wave = (uint32_t)__builtin_amdgcn_readfirstlane(threadIdx.x / 64), pieces = (cols + kN - 1) / kN;
  const uint32_t t = blockIdx.x / parts, part = blockIdx.x - t * parts, first = part * 256 + threadIdx.x;
  uint32_t key[kKeys], of[4], place[4] = {0, 0, 0, 0};
#pragma unroll
  for (uint32_t j = 0; j < 4; j++) of[j] = (uint32_t)ids[t * K + min(wave + 4 * j, K - 1)];
  const auto keys = [&](uint32_t i0) {
#pragma unroll
    for (uint32_t j = 0; j < kKeys; j++) {
      if (i0 + j * 64 >= A) break;
      key[j] = (uint32_t)ids[min(i0 + j * 64 + lane, A - 1)];
    }
  };
  keys(0);
  Few<kType, kN> v;
  if (first < pieces) v.load(x + t * x_stride + min(first * kN, cols - kN));
#pragma unroll
  for (uint32_t j = 0; j < 4; j++) loaded<true>(of[j]);
  // An assignment's place: how many keys (expert, then assignment; past the last id the largest) are below its own.
#pragma unroll 1
  for (uint32_t i0 = 0; i0 < A; i0 += 64 * kKeys) {
#pragma unroll
    for (uint32_t j = 0; j < kKeys; j++) {
      if (i0 + j * 64 >= A) break;
      key[j] = i0 + j * 64 + lane < A ? min(key[j], E) * kKey + i0 + j * 64 + lane : ~0u;
    }
#pragma unroll
    for (uint32_t i = 0; i < 4; i++) {
      if (wave + 4 * i >= K) break;
      const uint32_t own = min(of[i], E) * kKey + t * K + wave + 4 * i;
#pragma unroll
      for (uint32_t j = 0; j < kKeys; j++) {
        if (i0 + j * 64 >= A) break;
        place[i] += (uint32_t)__popcll(__ballot(key[j] < own));
      }
    }
    keys(i0 + 64 * kKeys);
  }
#pragma unroll
  for (uint32_t i = 0; i < 4; i++) {
    const uint32_t k = wave + 4 * i, a = t * K + k;
    if (k >= K) break;
    if (lane == 0) {
      const bool there = of[i] < E;
      places[k] = there ? place[i] : ~0u;
      if (part == 0) {
        out.places[a] = there ? (int32_t)place[i] : -1;
        if (there) out.order[place[i]] = (int32_t)a;
      }
    }
  }
  __syncthreads();
  uint32_t to[16];
#pragma unroll
  for (uint32_t k = 0; k < 16; k++) to[k] = (uint32_t)__builtin_amdgcn_readfirstlane((int)places[k]);
#pragma unroll 1
  for (uint32_t piece = first; piece < pieces; piece += parts * 256) {
    const uint32_t c = min(piece * kN, cols - kN);
    if (piece != first) v.load(x + t * x_stride + c);
#pragma unroll
    for (uint32_t k = 0; k < 16; k++)
      if (k < K && to[k] != ~0u) v.store(xs + (uint64_t)to[k] * xs_stride + c);
  }
}

// A token's rows, eight ranks' loads on their way at a time; each rank's product is fused into the sum, in rank order. A: rows of o.
template <bool kWide, uint32_t kIn, uint32_t kOut, uint32_t kN>
__global__ void __launch_bounds__(256) combine_rows(const typename Elem<kIn>::T *__restrict__ o, uint64_t o_stride, uint32_t A,
                                                    uint32_t ntok, uint32_t K, uint32_t cols, const int32_t *__restrict__ places,
                                                    const float *__restrict__ w, typename Elem<kOut>::T *__restrict__ y,
                                                    uint64_t y_stride) {
  each_piece<kWide, kN>(ntok, cols, [&](uint32_t t, uint32_t c) {
    float s[kN];
#pragma unroll
    for (uint32_t j = 0; j < kN; j++) s[j] = 0.0f;
#pragma unroll
    for (uint32_t k0 = 0; k0 < 16; k0 += 8) {
      if (k0 >= K) break;
      Few<kIn, kN> v[8];
      float f[8];
      uint32_t p[8];
#pragma unroll
      for (uint32_t k = 0; k < 8; k++) {
        const uint32_t a = t * K + min(k0 + k, K - 1);
        p[k] = (uint32_t)places[a];
        f[k] = w ? w[a] : 1.0f;
      }
#pragma unroll
      for (uint32_t k = 0; k < 8; k++) {
        loaded<kWide>(p[k]), loaded<kWide>(f[k]);
        if (k0 + k >= K) p[k] = ~0u;
      }
#pragma unroll
      for (uint32_t k = 0; k < 8; k++)
        if (p[k] < A) v[k].load(o + p[k] * o_stride + c);
#pragma unroll
      for (uint32_t k = 0; k < 8; k++)
        if (p[k] < A)
#pragma unroll
          for (uint32_t j = 0; j < kN; j++) s[j] = __builtin_fmaf(f[k], v[k][j], s[j]);
    }
    typedef typename Elem<kOut>::T T;
    if constexpr (kN == 1) {
      y[t * y_stride + c] = (T)s[0];
    } else {
      struct __attribute__((packed, aligned(sizeof(T)))) Pack {
        T e[kN];
      } r;
#pragma unroll
      for (uint32_t j = 0; j < kN; j++) r.e[j] = (T)s[j];
      *(Pack *)(y + t * y_stride + c) = r;
    }
  });
}

// A wave an assignment: do = w dy (in fp32, then rounded to the type) and dw = <dy, o>, four pieces of both rows on their way at a
// time; a lane's products are added in column order by their place in a piece, these sums and the lanes' by halves. dw or dout may be
// null. A row is one wave's whatever its length and the number of rows: 10 x 4096 of 64 bf16 values 17.4 us with the dispatch's
// gradient, one of 16384 fp32 values 22 us, one of 2^20 1.4 ms.
template <uint32_t kType, uint32_t kN>
__global__ void __launch_bounds__(256) combine_gradient(const typename Elem<kType>::T *__restrict__ dy, uint64_t dy_stride, uint32_t A,
                                                        uint32_t K, uint32_t cols, const int32_t *__restrict__ places,
                                                        const typename Elem<kType>::T *__restrict__ o, uint64_t o_stride,
                                                        const float *__restrict__ w, typename Elem<kType>::T *__restrict__ dout,
                                                        uint64_t do_stride, float *__restrict__ dw) {
  constexpr uint32_t kRun = 64 * kN;
  const uint32_t lane = threadIdx.x & 63, a = blockIdx.x * 4 + (uint32_t)__builtin_amdgcn_readfirstlane(threadIdx.x / 64);
  if (a >= A) return;
  const uint32_t p = (uint32_t)places[a];
  if (p >= A) {
    if (dw && lane == 0) dw[a] = 0.0f;
    return;
  }
  const float f = w ? w[a] : 1.0f;
  dy += a / K * dy_stride;
  if (dw) o += p * o_stride;
  if (dout) dout += p * do_stride;
  float s[kN];
#pragma unroll
  for (uint32_t n = 0; n < kN; n++) s[n] = 0.0f;
  for (uint32_t c0 = lane * kN; c0 < cols; c0 += 4 * kRun) {
    Few<kType, kN> d[4], v[4];
#pragma unroll
    for (uint32_t j = 0; j < 4; j++) {
      const uint32_t c = c0 + j * kRun;
      if (c >= cols) break;
      d[j].v = *(const typename Few<kType, kN>::V *)(dy + min(c, cols - kN));  // (read again by the token's other ranks)
      if (dw) v[j].load(o + min(c, cols - kN));
    }
#pragma unroll
    for (uint32_t j = 0; j < 4; j++) {
      const uint32_t c = c0 + j * kRun, at = min(c, cols - kN);
      if (c >= cols) break;
      if (dw)
#pragma unroll
        for (uint32_t n = 0; n < kN; n++)
          if (at + n >= c) s[n] = __builtin_fmaf(d[j][n], v[j][n], s[n]);  // (the others are the piece before's)
      if (dout) {
        float e[kN];
#pragma unroll
        for (uint32_t n = 0; n < kN; n++) e[n] = f * d[j][n];
        Few<kType, kN>::of(e).store(dout + at);
      }
    }
  }
  if (dw) {
#pragma unroll
    for (uint32_t m = kN / 2; m >= 1; m /= 2)
#pragma unroll
      for (uint32_t n = 0; n < m; n++) s[n] += s[n + m];
#pragma unroll
    for (uint32_t m = 32; m >= 1; m /= 2) s[0] += __shfl_xor(s[0], (int)m, 64);
    if (lane == 0) dw[a] = s[0];
  }
}

// ---- host

namespace {

// f(whether the rows' pieces are wide, the elements of a piece) as constants, for rows of kType: waves of one row's pieces where
// that leaves no more than half of the lanes without one.
template <uint32_t kType, typename F>
void op_by_pieces(uint32_t cols, F f) {
  constexpr uint32_t kN = kWhole<kType>;
  if (cols >= 32 * kN) return f(std::true_type(), std::integral_constant<uint32_t, kN>());
  if (cols >= kN) return f(std::false_type(), std::integral_constant<uint32_t, kN>());
  f(std::false_type(), std::integral_constant<uint32_t, 1>());
}
// launch(t0, tokens, work-groups) for as many tokens at a time as a launch has threads for.
template <typename F>
void by_tokens(uint32_t ntok, bool wide, uint32_t pieces, F launch) {
  const uint32_t runs = (pieces + 63) / 64, most = wide ? (1u << 25) / runs : ntok;
  for (uint32_t t0 = 0; t0 < ntok; t0 += most) {
    const uint32_t n = std::min(ntok - t0, most);
    launch(t0, n, wide ? ((uint64_t)n * runs + 3) / 4 : ((uint64_t)n * pieces + 255) / 256);
  }
}

}  // namespace

uint64_t sort_bytes(uint32_t A, uint32_t E) { return slices_of(A) > 1 ? (uint64_t)slices_of(A) * E * 4 : 0; }

void sort_launch(const int32_t *ids, uint32_t A, uint32_t E, const SortOut &out, void *work, void *stream) {
  const uint32_t slice = slice_of(A), slices = slices_of(A);
  uint32_t *counts = (uint32_t *)work;
  if (slices > 1) op_launch(sort_count, slices, 1024, stream, ids, A, E, slice, counts);
  sort_place_launch(ids, A, E, out, work, stream);
}

void sort_place_launch(const int32_t *ids, uint32_t A, uint32_t E, const SortOut &out, void *work, void *stream) {
  const uint32_t slice = slice_of(A), slices = slices_of(A);
  uint32_t *counts = (uint32_t *)work;
  if (slice == kSlice)
    op_launch(sort_place<true>, slices, 64 * kSortWaves, stream, ids, A, E, slice, (const uint32_t *)counts, out);
  else
    op_launch(sort_place<false>, slices, 64 * kSortWaves, stream, ids, A, E, slice, (const uint32_t *)counts, out);
}

void combine_launch(uint32_t type, const void *o, uint64_t o_stride, uint32_t ntok, uint32_t K, uint32_t cols,
                    const int32_t *places, const float *w, uint32_t y_type, void *y, uint64_t y_stride, void *stream) {
  op_by_type(type, [&](auto in) {
    op_by_type(y_type, [&](auto out) {
      constexpr uint32_t kIn = decltype(in)::value, kOut = decltype(out)::value;
      if constexpr (kIn == QT_F32 || kIn == kOut) {
        op_by_pieces<kIn>(cols, [&](auto wide, auto piece) {
          constexpr bool kWide = decltype(wide)::value;
          constexpr uint32_t kN = decltype(piece)::value;
          by_tokens(ntok, kWide, (cols + kN - 1) / kN, [&](uint32_t t0, uint32_t n, uint64_t blocks) {
            op_launch(combine_rows<kWide, kIn, kOut, kN>, blocks, 256, stream, (const typename Elem<kIn>::T *)o, o_stride, ntok * K, n,
                      K, cols, places + (uint64_t)t0 * K, w ? w + (uint64_t)t0 * K : nullptr,
                      (typename Elem<kOut>::T *)y + t0 * y_stride, y_stride);
          });
        });
      }
    });
  });
}

}  // namespace c0ven

using namespace c0ven;

namespace {

constexpr uint32_t kMostTokens = 1u << 20;

void check_dispatch(const moe_dispatch_config *c, uint32_t ntok) {
  op_require(c != nullptr, "null argument");
  op_require(c->n_expert >= 1 && c->n_expert <= kMostExperts, "n_expert must be 1..512");
  op_require(c->n_used >= 1 && c->n_used <= 16, "n_used must be 1..16");
  op_require(c->n_embd >= 1 && c->n_embd <= 1u << 20, "n_embd must be 1..2^20");
  op_require(op_float(c->type), "the element type must be QT_F32, QT_F16 or QT_BF16");
  op_require(ntok <= kMostTokens, "at most 2^20 tokens");
}
void op_words(const void *p, uint32_t ntok, const char *why) { op_require((p || !ntok) && op_aligned(p, 4), why); }

}  // namespace

extern "C" {

MOE_API uint64_t moe_dispatch_work_bytes(const moe_dispatch_config *cfg, uint32_t ntok) {
  uint64_t n = 0;
  (void)op_guarded([&] {
    check_dispatch(cfg, ntok);
    n = sort_bytes(ntok * cfg->n_used, cfg->n_expert);
  });
  return n;
}

MOE_API moe_status moe_dispatch_async(const moe_dispatch_config *cfg, const void *x, uint64_t x_stride, uint32_t ntok,
                                      const int32_t *ids, void *xs, uint64_t xs_stride, int32_t *order, int32_t *places,
                                      uint32_t *offsets, void *work, uint64_t work_bytes, void *stream) {
  return op_guarded([&] {
    check_dispatch(cfg, ntok);
    const uint32_t H = cfg->n_embd, K = cfg->n_used, E = cfg->n_expert, A = ntok * K, size = op_size(cfg->type);
    if (xs) {
      op_rows(x, x_stride, ntok, H, cfg->type);
      op_rows(xs, xs_stride, ntok, H, cfg->type);
    }
    op_words(ids, ntok, "null or misaligned ids");
    op_words(order, ntok, "null or misaligned order");
    op_words(places, ntok, "null or misaligned places");
    op_require(offsets && op_aligned(offsets, 4), "null or misaligned offsets");
    op_work(work, work_bytes, sort_bytes(A, E));
    OnDevice on(cfg->device);
    const SortOut out{order, places, offsets, nullptr, nullptr, 1};
    if (A > kFewIds) sort_launch(ids, A, E, out, work, stream);
    // (Copies: the element type matters by its size alone.)
    const auto rows = [&](auto t) {
      constexpr uint32_t kType = decltype(t)::value;
      const auto *from = (const typename Elem<kType>::T *)x;
      auto *to = (typename Elem<kType>::T *)xs;
      op_by_pieces<kType>(H, [&](auto wide, auto piece) {
        constexpr bool kWide = decltype(wide)::value;
        constexpr uint32_t kN = decltype(piece)::value;
        if (A <= kFewIds) {
          const uint32_t cols = xs ? H : 0;
          // (More than 1024 work-groups would only read the ids more often.)
          const uint32_t most = std::max(((cols + kN - 1) / kN + 255) / 256, 1u);
          const uint32_t parts = std::min(most, std::max(1024 / std::max(ntok, 1u), 1u));
          return op_launch(dispatch_few<kType, kN>, (uint64_t)ntok * parts + 1, 256, stream, ids, ntok, K, E, from, x_stride, cols, to,
                           xs_stride, parts, out);
        }
        if (!xs) return;
        by_tokens(ntok, kWide, (H + kN - 1) / kN, [&](uint32_t t0, uint32_t n, uint64_t blocks) {
          op_launch(dispatch_rows<kWide, kType, kN>, blocks, 256, stream, from + t0 * x_stride, x_stride, n, K, H,
                    (const int32_t *)places + (uint64_t)t0 * K, to, xs_stride);
        });
      });
    };
    if (size == 4)
      rows(std::integral_constant<uint32_t, QT_F32>());
    else
      rows(std::integral_constant<uint32_t, QT_F16>());
  });
}

MOE_API moe_status moe_combine_async(const moe_dispatch_config *cfg, const void *o, uint64_t o_stride, uint32_t ntok,
                                     const int32_t *places, const float *w, void *y, uint64_t y_stride, void *stream) {
  return op_guarded([&] {
    check_dispatch(cfg, ntok);
    op_rows(o, o_stride, ntok, cfg->n_embd, cfg->type);
    op_rows(y, y_stride, ntok, cfg->n_embd, cfg->type);
    op_words(places, ntok, "null or misaligned places");
    op_require(op_aligned(w, 4), "misaligned w");
    if (!ntok) return;
    OnDevice on(cfg->device);
    combine_launch(cfg->type, o, o_stride, ntok, cfg->n_used, cfg->n_embd, places, w, cfg->type, y, y_stride, stream);
  });
}

MOE_API moe_status moe_dispatch_backward_async(const moe_dispatch_config *cfg, const void *dxs, uint64_t dxs_stride, uint32_t ntok,
                                               const int32_t *places, void *dx, uint64_t dx_stride, void *stream) {
  return moe_combine_async(cfg, dxs, dxs_stride, ntok, places, nullptr, dx, dx_stride, stream);
}

MOE_API moe_status moe_combine_backward_async(const moe_dispatch_config *cfg, const void *dy, uint64_t dy_stride, uint32_t ntok,
                                              const int32_t *places, const void *o, uint64_t o_stride, const float *w, void *dout,
                                              uint64_t dout_stride, float *dw, void *stream) {
  return op_guarded([&] {
    check_dispatch(cfg, ntok);
    const uint32_t H = cfg->n_embd, K = cfg->n_used, A = ntok * K;
    op_rows(dy, dy_stride, ntok, H, cfg->type);
    op_words(places, ntok, "null or misaligned places");
    op_require(op_aligned(w, 4) && op_aligned(dw, 4), "misaligned w or dw");
    if (dw) op_rows(o, o_stride, ntok, H, cfg->type);
    if (dout) op_rows(dout, dout_stride, ntok, H, cfg->type);
    if (!ntok || (!dw && !dout)) return;
    OnDevice on(cfg->device);
    op_by_type(cfg->type, [&](auto t) {
      constexpr uint32_t kType = decltype(t)::value;
      typedef typename Elem<kType>::T T;
      op_by_pieces<kType>(H, [&](auto, auto piece) {
        op_launch(combine_gradient<kType, decltype(piece)::value>, ((uint64_t)A + 3) / 4, 256, stream, (const T *)dy, dy_stride, A, K, H,
                  places, (const T *)o, o_stride, w, (T *)dout, dout_stride, dw);
      });
    });
  });
}

}  // extern "C"
