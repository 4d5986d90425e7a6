// Tokens sorted by expert and back (moe_dispatch_async, moe_combine_async) and the gradients of both.
//
// All of it moves rows: bound by memory. The sort is a stable counting sort of the ids; the rows are read and written 16 bytes
// a lane, a wave a run of 64 such pieces of one token, whose places are then the wave's (scalar loads).
#include "dispatch.h"
#include "experts.h"
#include "mx4_api.h"

#include <algorithm>

namespace c0ven {

// ---- the sort

constexpr uint32_t kSlice = 4096;     // ids a work-group sorts, at least
constexpr uint32_t kMostSlices = 256; // (each work-group reads all slices' counts)
constexpr uint32_t kMostExperts = 512;
constexpr uint32_t kSortWaves = 16;

// counts[slice][expert] of `slice` ids each.
__global__ void __launch_bounds__(1024) sort_count(const int32_t *ids, uint32_t A, uint32_t E, uint32_t slice, uint32_t *counts) {
  __shared__ uint32_t n[kMostExperts];
  const uint32_t first = blockIdx.x * slice, end = min(A, first + slice);
  if (threadIdx.x < kMostExperts) n[threadIdx.x] = 0;
  __syncthreads();
  for (uint32_t i0 = first + threadIdx.x; i0 < end; i0 += 4 * 1024) {
    uint32_t id[4];
#pragma unroll
    for (uint32_t j = 0; j < 4; j++) id[j] = i0 + j * 1024 < end ? (uint32_t)ids[i0 + j * 1024] : ~0u;
#pragma unroll
    for (uint32_t j = 0; j < 4; j++)
      if (id[j] < E) atomicAdd(n + id[j], 1u);
  }
  __syncthreads();
  if (threadIdx.x < E) counts[blockIdx.x * E + threadIdx.x] = n[threadIdx.x];
}

// The places of a slice's assignments: an expert's start, its assignments in the slices before, those of the waves before (each
// has a sixteenth of the slice) and, 64 ids at a time, those of the lanes before. Equal ids keep their order, so equal calls
// give equal places.
__global__ void __launch_bounds__(64 * kSortWaves) sort_place(const int32_t *ids, uint32_t A, uint32_t E, uint32_t slice,
                                                              const uint32_t *counts, SortOut out) {
  __shared__ uint32_t at[kSortWaves][kMostExperts];
  __shared__ uint32_t half[2][kMostExperts];
  __shared__ uint32_t sums[2][8];
  __shared__ uint32_t total;
  const uint32_t tid = threadIdx.x, lane = tid & 63, wave = tid / 64, bits = 32 - (uint32_t)__clz((int)((E - 1) | 1));
  const uint32_t first = blockIdx.x * slice, end = min(A, first + slice);
  const uint32_t run = slice / kSortWaves, from = min(first + wave * run, end), to = min(from + run, end);
  for (uint32_t i = tid; i < kSortWaves * kMostExperts; i += 64 * kSortWaves) at[0][i] = 0;
  __syncthreads();
  for (uint32_t i0 = from + lane; i0 < to; i0 += 4 * 64) {
    uint32_t id[4];
#pragma unroll
    for (uint32_t j = 0; j < 4; j++) id[j] = i0 + j * 64 < to ? (uint32_t)ids[i0 + j * 64] : ~0u;
#pragma unroll
    for (uint32_t j = 0; j < 4; j++)
      if (id[j] < E) atomicAdd(&at[wave][id[j]], 1u);
  }
  // An expert's assignments in all slices and in those before: two threads an expert, every second slice each.
  const uint32_t e = tid % kMostExperts, h = tid / kMostExperts;
  uint32_t all = 0, before = 0;
  if (gridDim.x > 1 && e < E)
    for (uint32_t s0 = h; s0 < gridDim.x; s0 += 16) {
      uint32_t c[8];
#pragma unroll
      for (uint32_t j = 0; j < 8; j++) c[j] = s0 + 2 * j < gridDim.x ? counts[(s0 + 2 * j) * E + e] : 0;
#pragma unroll
      for (uint32_t j = 0; j < 8; j++) all += c[j], before += s0 + 2 * j < blockIdx.x ? c[j] : 0;
    }
  if (h == 1) half[0][e] = all, half[1][e] = before;
  __syncthreads();
  uint32_t own = 0, tiles = 0;
  if (h == 0) {
    all += half[0][e], before += half[1][e];
    for (uint32_t v = 0; v < kSortWaves; v++) {
      const uint32_t n = at[v][e];
      at[v][e] = own;
      own += n;
    }
    if (gridDim.x == 1) all = own;
    if (out.tiles) tiles = (all + out.rows - 1) / out.rows;
  }
  uint32_t place = all, tile = tiles;  // their sums up to this expert
  for (uint32_t d = 1; d < 64; d *= 2) {
    const uint32_t p = (uint32_t)__shfl_up((int)place, d, 64), t = (uint32_t)__shfl_up((int)tile, d, 64);
    if (lane >= d) place += p, tile += t;
  }
  if (h == 0 && lane == 63) sums[0][wave] = place, sums[1][wave] = tile;
  __syncthreads();
  if (h == 0) {
    for (uint32_t v = 0; v < wave; v++) place += sums[0][v], tile += sums[1][v];
    for (uint32_t v = 0; v < kSortWaves; v++) at[v][e] += place - all + before;
    if (e == kMostExperts - 1) total = place;
    if (blockIdx.x == 0) {
      if (e < E) out.offsets[e] = place - all;
      if (e == E - 1) out.offsets[E] = place;
      if (out.tiles) {
        for (uint32_t j = 0; j < tiles; j++)
          out.tiles[tile - tiles + j] = MoeTile{e, e, place - all + j * out.rows, min(out.rows, all - j * out.rows)};
        if (e == kMostExperts - 1) *out.n_tiles = tile;
      }
    }
  }
  __syncthreads();
  for (uint32_t i0 = from; i0 < to; i0 += 64) {
    const uint32_t i = i0 + lane, id = i < to ? (uint32_t)ids[i] : ~0u;
    const bool in = id < E;
    uint64_t same = __ballot(in);
    for (uint32_t b = 0; b < bits; b++) {
      const uint64_t set = __ballot(id >> b & 1);
      same &= id >> b & 1 ? set : ~set;
    }
    if (in) {
      const uint32_t under = lanes_below(same), p = at[wave][id] + under;
      if (under == 0) at[wave][id] = p + (uint32_t)__popcll(same);
      out.order[p] = (int32_t)i;
      out.places[i] = (int32_t)p;
    } else if (i < to) {
      out.places[i] = -1;
    }
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");  // (the counts before the next ids')
    __builtin_amdgcn_wave_barrier();
  }
  for (uint32_t i = max(first, total) + tid; i < end; i += 64 * kSortWaves) out.order[i] = -1;
}

// ---- rows out

// 16 bytes of a row at whatever address (or what is left of it), two at a time at the end (rows are of whole elements).
struct __attribute__((packed, aligned(2))) Piece {
  uint16_t v[8];
};
__device__ __forceinline__ Piece piece_of(const uint8_t *row, uint64_t at, uint64_t n) {
  if (at + 16 <= n) return *(const Piece *)(row + at);
  Piece p = {};
#pragma unroll
  for (uint32_t j = 0; j < 8; j++)
    if (at + 2 * j < n) p.v[j] = *(const uint16_t *)(row + at + 2 * j);
  return p;
}
__device__ __forceinline__ void put_piece(uint8_t *row, uint64_t at, uint64_t n, const Piece &p) {
  if (at + 16 <= n) {
    *(Piece *)(row + at) = p;
    return;
  }
#pragma unroll
  for (uint32_t j = 0; j < 8; j++)
    if (at + 2 * j < n) *(uint16_t *)(row + at + 2 * j) = p.v[j];
}

// Which token and which piece (of `per` a row) a lane has: kWide: a wave's 64 pieces are one token's, so that what goes by the
// token is scalar (rows of at least 32 pieces); else the lanes follow one another through the rows.
constexpr uint32_t kWidePieces = 32;
template <bool kWide>
struct Items {
  uint64_t n;     // waves (kWide) or lanes
  uint32_t per;
  __host__ __device__ Items(uint64_t rows, uint32_t pieces) : n(rows * (kWide ? (pieces + 63) / 64 : pieces)), per(pieces) {}
  __host__ __device__ uint64_t blocks() const { return (n + (kWide ? 3 : 255)) / (kWide ? 4 : 256); }
  // f(row, piece) of block b's lanes.
  template <typename F>
  __device__ __forceinline__ void each(uint64_t b, F f) const {
    if (kWide) {
      const uint32_t runs = (per + 63) / 64;
      const uint64_t item = b * 4 + (uint32_t)__builtin_amdgcn_readfirstlane(threadIdx.x / 64);
      if (item >= n) return;
      const uint32_t row = (uint32_t)(item / runs), piece = (uint32_t)(item - (uint64_t)row * runs) * 64 + threadIdx.x % 64;
      if (piece < per) f(row, piece);
    } else {
      const uint64_t i = b * 256 + threadIdx.x;
      if (i >= n) return;
      const uint32_t row = (uint32_t)(i / per);
      f(row, (uint32_t)(i - (uint64_t)row * per));
    }
  }
};
// Work-groups of a launch: as many as there are items, or what goes through them in turn.
constexpr uint64_t kMostBlocks = 1 << 20;

// Each token's row to its ranks' places.
template <bool kWide>
__global__ void __launch_bounds__(256) dispatch_rows(const uint8_t *x, uint64_t x_stride, uint32_t ntok, uint32_t K, uint64_t bytes,
                                                     const int32_t *places, uint8_t *xs, uint64_t xs_stride) {
  const Items<kWide> items(ntok, (uint32_t)((bytes + 15) / 16));
  for (uint64_t b = blockIdx.x; b < items.blocks(); b += gridDim.x)
    items.each(b, [&](uint32_t t, uint32_t piece) {
      const Piece p = piece_of(x + t * x_stride, (uint64_t)piece * 16, bytes);
      int32_t to[16];
#pragma unroll
      for (uint32_t k = 0; k < 16; k++) to[k] = k < K ? places[(uint64_t)t * K + k] : -1;
#pragma unroll
      for (uint32_t k = 0; k < 16; k++)
        if (to[k] >= 0) put_piece(xs + (uint64_t)(uint32_t)to[k] * xs_stride, (uint64_t)piece * 16, bytes, p);
    });
}

// At most kFewIds ids: the sort and the rows in one launch, each wave counting its token's places itself (those of lower ids and
// of equal ones before), the last work-group the offsets. bytes 0: no rows.
constexpr uint32_t kFewIds = 1024;
__global__ void __launch_bounds__(256) dispatch_few(const int32_t *ids, uint32_t ntok, uint32_t K, uint32_t E, const uint8_t *x,
                                                    uint64_t x_stride, uint64_t bytes, uint8_t *xs, uint64_t xs_stride, SortOut out) {
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
  uint32_t id[kFewIds / 64];
#pragma unroll
  for (uint32_t j = 0; j < kFewIds / 64; j++) id[j] = j * 64 + lane < A ? min((uint32_t)ids[j * 64 + lane], E) : E;
  const uint32_t pieces = (uint32_t)((bytes + 15) / 16), runs = max((pieces + 63) / 64, 1u);
  const uint64_t item = (uint64_t)blockIdx.x * 4 + (uint32_t)__builtin_amdgcn_readfirstlane(threadIdx.x / 64);
  if (item >= (uint64_t)ntok * runs) return;
  const uint32_t t = (uint32_t)(item / runs), run = (uint32_t)(item - (uint64_t)t * runs), piece = run * 64 + lane;
  const Piece p = piece < pieces ? piece_of(x + t * x_stride, (uint64_t)piece * 16, bytes) : Piece{};
  for (uint32_t k = 0; k < K; k++) {
    const uint32_t a = t * K + k, e = min((uint32_t)ids[a], E);
    uint32_t place = 0;
#pragma unroll
    for (uint32_t j = 0; j < kFewIds / 64; j++) {
      if (j * 64 >= A) break;
      place += (uint32_t)__popcll(__ballot(id[j] < e || (id[j] == e && j * 64 + lane < a)));
    }
    if (run == 0 && lane == 0) {
      out.places[a] = e < E ? (int32_t)place : -1;
      if (e < E) out.order[place] = (int32_t)a;
    }
    if (e < E && piece < pieces) put_piece(xs + (uint64_t)place * xs_stride, (uint64_t)piece * 16, bytes, p);
  }
}

// ---- rows back

// 16 bytes of elements, as they lie in memory.
template <uint32_t kType>
struct Few {
  static constexpr uint32_t kN = 16 / sizeof(typename Elem<kType>::T);
  typedef typename Elem<kType>::T T;
  struct __attribute__((packed)) Pack {
    T e[kN];
  } p;
  // Those from column c on (zeros past a row's end).
  __device__ __forceinline__ void load(const T *row, uint32_t c, uint32_t cols) {
    if (c + kN <= cols) {
      p = *(const Pack *)(row + c);
    } else {
#pragma unroll
      for (uint32_t j = 0; j < kN; j++) p.e[j] = c + j < cols ? row[c + j] : (T)0.0f;
    }
  }
  __device__ __forceinline__ float operator[](uint32_t j) const { return (float)p.e[j]; }
};
template <uint32_t kType, uint32_t kN>
__device__ __forceinline__ void store_few(typename Elem<kType>::T *row, uint32_t c, uint32_t cols, const float v[kN]) {
  typedef typename Elem<kType>::T T;
  struct __attribute__((packed)) Pack {
    T e[kN];
  };
  if (c + kN <= cols) {
    Pack p;
#pragma unroll
    for (uint32_t j = 0; j < kN; j++) p.e[j] = (T)v[j];
    *(Pack *)(row + c) = p;
  } else {
#pragma unroll
    for (uint32_t j = 0; j < kN; j++)
      if (c + j < cols) row[c + j] = (T)v[j];
  }
}

// A token's rows, eight ranks' loads on their way at a time; each rank's product is fused into the sum, in rank order.
template <bool kWide, uint32_t kIn, uint32_t kOut>
__global__ void __launch_bounds__(256) combine_rows(const typename Elem<kIn>::T *o, uint64_t o_stride, uint32_t ntok, uint32_t K,
                                                    uint32_t cols, const int32_t *places, const float *w,
                                                    typename Elem<kOut>::T *y, uint64_t y_stride) {
  constexpr uint32_t kN = Few<kIn>::kN;
  const uint32_t A = ntok * K;
  const Items<kWide> items(ntok, (cols + kN - 1) / kN);
  for (uint64_t b = blockIdx.x; b < items.blocks(); b += gridDim.x)
    items.each(b, [&](uint32_t t, uint32_t piece) {
      float s[kN];
#pragma unroll
      for (uint32_t j = 0; j < kN; j++) s[j] = 0.0f;
#pragma unroll
      for (uint32_t k0 = 0; k0 < 16; k0 += 8) {
        if (k0 >= K) break;
        Few<kIn> v[8];
        float f[8];
        bool on[8];
#pragma unroll
        for (uint32_t k = 0; k < 8; k++) {
          const uint32_t a = t * K + min(k0 + k, K - 1), p = (uint32_t)places[a];
          on[k] = k0 + k < K && p < A;
          f[k] = w ? w[a] : 1.0f;
          if (on[k]) v[k].load(o + p * o_stride, piece * kN, cols);
        }
#pragma unroll
        for (uint32_t k = 0; k < 8; k++)
          if (on[k])
#pragma unroll
            for (uint32_t j = 0; j < kN; j++) s[j] = __builtin_fmaf(f[k], v[k][j], s[j]);
      }
      store_few<kOut, kN>(y + t * y_stride, piece * kN, cols, s);
    });
}

// A wave an assignment: do = w dy (rounded once) and dw = <dy, o>, four pieces of both rows on their way at a time; a lane's
// products are added in column order, the lanes' sums by halves. dw or dout may be null.
template <uint32_t kType>
__global__ void __launch_bounds__(256) combine_gradient(const typename Elem<kType>::T *dy, uint64_t dy_stride, uint32_t A, uint32_t K,
                                                        uint32_t cols, const int32_t *places, const typename Elem<kType>::T *o,
                                                        uint64_t o_stride, const float *w, typename Elem<kType>::T *dout,
                                                        uint64_t do_stride, float *dw) {
  constexpr uint32_t kN = Few<kType>::kN, kRun = 64 * kN;
  const uint32_t lane = threadIdx.x & 63;
  for (uint64_t i = (uint64_t)blockIdx.x * 4; i < A; i += (uint64_t)gridDim.x * 4) {
    const uint32_t a = (uint32_t)i + (uint32_t)__builtin_amdgcn_readfirstlane(threadIdx.x / 64);
    if (a >= A) continue;
    const uint32_t p = (uint32_t)places[a];
    if (p >= A) {
      if (dw && lane == 0) dw[a] = 0.0f;
      continue;
    }
    const float f = w ? w[a] : 1.0f;
    const auto *from = dy + (uint64_t)(a / K) * dy_stride;
    float s = 0.0f;
    for (uint32_t c0 = lane * kN; c0 < cols; c0 += 4 * kRun) {
      Few<kType> d[4], v[4];
#pragma unroll
      for (uint32_t j = 0; j < 4; j++) {
        const uint32_t c = c0 + j * kRun;
        if (c >= cols) break;
        d[j].load(from, c, cols);
        if (dw) v[j].load(o + p * o_stride, c, cols);
      }
#pragma unroll
      for (uint32_t j = 0; j < 4; j++) {
        const uint32_t c = c0 + j * kRun;
        if (c >= cols) break;
        if (dw)
#pragma unroll
          for (uint32_t n = 0; n < kN; n++) s = __builtin_fmaf(d[j][n], v[j][n], s);
        if (dout) {
          float e[kN];
#pragma unroll
          for (uint32_t n = 0; n < kN; n++) e[n] = f * d[j][n];
          store_few<kType, kN>(dout + p * do_stride, c, cols, e);
        }
      }
    }
    if (dw) {
#pragma unroll
      for (uint32_t m = 32; m >= 1; m /= 2) s += __shfl_xor(s, (int)m, 64);
      if (lane == 0) dw[a] = s;
    }
  }
}

// ---- host

namespace {

uint32_t slice_of(uint32_t A) {
  const uint32_t n = (A + kSlice - 1) / kSlice;
  return kSlice * ((n + kMostSlices - 1) / kMostSlices);
}
uint32_t slices_of(uint32_t A) { return A ? (A + slice_of(A) - 1) / slice_of(A) : 0; }

// f with whether the rows' pieces are wide, as a constant.
template <typename F>
void op_by_width(uint64_t pieces, F f) {
  if (pieces >= kWidePieces)
    f(std::true_type());
  else
    f(std::false_type());
}

}  // namespace

uint64_t sort_bytes(uint32_t A, uint32_t E) { return slices_of(A) > 1 ? (uint64_t)slices_of(A) * E * 4 : 0; }

void sort_launch(const int32_t *ids, uint32_t A, uint32_t E, const SortOut &out, void *work, void *stream) {
  const uint32_t slice = slice_of(A), slices = slices_of(A);
  uint32_t *counts = (uint32_t *)work;
  if (slices > 1) op_launch(sort_count, slices, 1024, stream, ids, A, E, slice, counts);
  op_launch(sort_place, slices, 64 * kSortWaves, stream, ids, A, E, slice, (const uint32_t *)counts, out);
}

void combine_launch(uint32_t type, const void *o, uint64_t o_stride, uint32_t ntok, uint32_t K, uint32_t cols,
                    const int32_t *places, const float *w, uint32_t y_type, void *y, uint64_t y_stride, void *stream) {
  op_by_type(type, [&](auto in) {
    op_by_type(y_type, [&](auto out) {
      constexpr uint32_t kIn = decltype(in)::value, kOut = decltype(out)::value;
      if constexpr (kIn == QT_F32 || kIn == kOut) {
        const uint32_t pieces = (cols + Few<kIn>::kN - 1) / Few<kIn>::kN;
        op_by_width(pieces, [&](auto wide) {
          constexpr bool kWide = decltype(wide)::value;
          const uint64_t n = std::min(Items<kWide>(ntok, pieces).blocks(), kMostBlocks);
          op_launch(combine_rows<kWide, kIn, kOut>, n, 256, stream, (const typename Elem<kIn>::T *)o, o_stride, ntok, K, cols, places,
                    w, (typename Elem<kOut>::T *)y, y_stride);
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
    const uint8_t *from = (const uint8_t *)x;
    uint8_t *to = (uint8_t *)xs;
    const uint64_t bytes = xs ? (uint64_t)H * size : 0, pieces = (bytes + 15) / 16;
    if (A <= kFewIds) {
      const uint64_t waves = ntok * std::max<uint64_t>((pieces + 63) / 64, 1);
      return op_launch(dispatch_few, (waves + 3) / 4 + 1, 256, stream, ids, ntok, K, E, from, x_stride * size, bytes, to,
                       xs_stride * size, out);
    }
    sort_launch(ids, A, E, out, work, stream);
    if (xs)
      op_by_width(pieces, [&](auto wide) {
        constexpr bool kWide = decltype(wide)::value;
        op_launch(dispatch_rows<kWide>, std::min(Items<kWide>(ntok, (uint32_t)pieces).blocks(), kMostBlocks), 256, stream, from,
                  x_stride * size, ntok, K, bytes, (const int32_t *)places, to, xs_stride * size);
      });
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
      typedef typename Elem<decltype(t)::value>::T T;
      op_launch(combine_gradient<decltype(t)::value>, std::min<uint64_t>(((uint64_t)A + 3) / 4, kMostBlocks), 256, stream,
                (const T *)dy, dy_stride, A, K, H, places, (const T *)o, o_stride, w, (T *)dout, dout_stride, dw);
    });
  });
}

}  // extern "C"
