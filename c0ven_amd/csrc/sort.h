// The stable counting sort of assignments by expert: a work-group's part of it.
#pragma once

#include "dispatch.h"
#include "experts.h"

namespace c0ven {

constexpr uint32_t kSlice = 4096;     // ids a work-group sorts, at least
constexpr uint32_t kMostSlices = 256; // (each work-group reads all slices' counts)
constexpr uint32_t kMostExperts = 512;
constexpr uint32_t kSortWaves = 16;

// counts[slice][expert] of `slice` ids each; 1024 threads, a work-group a slice from the first on (place_slice too).
__device__ __forceinline__ void count_slice(const int32_t *ids, uint32_t A, uint32_t E, uint32_t slice, uint32_t *counts) {
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
// give equal places. kOnce: a slice of kSlice ids, which stay in registers with their ranks within the wave (3996 ids 6.5 us with
// a pass of atomics for the counts and the ids loaded again one step at a time).
template <bool kOnce>
__device__ __forceinline__ void place_slice(const int32_t *ids, uint32_t A, uint32_t E, uint32_t slice, uint32_t slices,
                                            const uint32_t *counts, const SortOut &out) {
  __shared__ __align__(16) uint32_t at[kSortWaves][kMostExperts];
  __shared__ uint32_t half[2][kMostExperts];
  __shared__ uint32_t sums[2][8];
  __shared__ uint32_t total;
  constexpr uint32_t kSteps = kSlice / kSortWaves / 64;
  const uint32_t tid = threadIdx.x, lane = tid & 63, wave = tid / 64, bits = 32 - (uint32_t)__clz((int)((E - 1) | 1));
  const uint32_t first = blockIdx.x * slice, end = min(A, first + slice);
  const uint32_t run = slice / kSortWaves, from = min(first + wave * run, end), to = min(from + run, end);
  uint32_t id[kSteps], rank[kSteps];
  if (kOnce)
#pragma unroll
    for (uint32_t j = 0; j < kSteps; j++) id[j] = from + j * 64 + lane < to ? (uint32_t)ids[from + j * 64 + lane] : ~0u;
  for (uint32_t i = tid; i < kSortWaves * kMostExperts / 4; i += 64 * kSortWaves) ((uint4 *)at)[i] = make_uint4(0, 0, 0, 0);
  // An expert's assignments in all slices and in those before: two threads an expert, every second slice each.
  const uint32_t e = tid % kMostExperts, h = tid / kMostExperts;
  uint32_t all = 0, before = 0;
  if (slices > 1 && e < E)
    for (uint32_t s0 = h; s0 < slices; s0 += 16) {
      uint32_t c[8];
#pragma unroll
      for (uint32_t j = 0; j < 8; j++) c[j] = counts[min(s0 + 2 * j, slices - 1) * E + e];
#pragma unroll
      for (uint32_t j = 0; j < 8; j++) {
        const uint32_t n = s0 + 2 * j < slices ? c[j] : 0;
        all += n, before += s0 + 2 * j < blockIdx.x ? n : 0;
      }
    }
  if (h == 1) half[0][e] = all, half[1][e] = before;
  __syncthreads();
  // 64 ids: what was counted of each one's expert before it; the counts go on.
  const auto count = [&](uint32_t x) {
    const bool in = x < E;
    uint64_t same = __ballot(in);
    for (uint32_t b = 0; b < bits; b++) {
      const uint64_t set = __ballot(x >> b & 1);
      same &= x >> b & 1 ? set : ~set;
    }
    uint32_t p = 0;
    if (in) {
      const uint32_t under = lanes_below(same);
      p = at[wave][x] + under;
      if (under == 0) at[wave][x] = p + (uint32_t)__popcll(same);
    }
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");  // (the counts before the next ids')
    __builtin_amdgcn_wave_barrier();
    return p;
  };
  if (kOnce) {
#pragma unroll
    for (uint32_t j = 0; j < kSteps; j++) rank[j] = count(id[j]);
  } else {
    for (uint32_t i0 = from; i0 < to; i0 += 64) (void)count(i0 + lane < to ? (uint32_t)ids[i0 + lane] : ~0u);
  }
  __syncthreads();
  uint32_t own = 0, tiles = 0, n[kSortWaves];
  if (h == 0) {
    all += half[0][e], before += half[1][e];
#pragma unroll
    for (uint32_t v = 0; v < kSortWaves; v++) n[v] = at[v][e];
#pragma unroll
    for (uint32_t v = 0; v < kSortWaves; v++) {
      const uint32_t m = n[v];
      n[v] = own;
      own += m;
    }
    if (slices == 1) all = own;
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
#pragma unroll
    for (uint32_t v = 0; v < kSortWaves; v++) at[v][e] = n[v] + place - all + before;
    if (e == kMostExperts - 1) total = place;
  }
  __syncthreads();
  const auto put = [&](uint32_t i, uint32_t x, uint32_t p) {
    if (x < E) {
      out.order[p] = (int32_t)i;
      out.places[i] = (int32_t)p;
    } else if (i < to) {
      out.places[i] = -1;
    }
  };
  if (kOnce) {
#pragma unroll
    for (uint32_t j = 0; j < kSteps; j++) put(from + j * 64 + lane, id[j], rank[j] + (id[j] < E ? at[wave][id[j]] : 0));
  } else {
    for (uint32_t i0 = from; i0 < to; i0 += 64) {
      const uint32_t x = i0 + lane < to ? (uint32_t)ids[i0 + lane] : ~0u;
      put(i0 + lane, x, count(x));
    }
  }
  for (uint32_t i = max(first, total) + tid; i < end; i += 64 * kSortWaves) out.order[i] = -1;
  if (blockIdx.x == 0 && h == 0) {
    if (e < E) out.offsets[e] = place - all;
    if (e == E - 1) out.offsets[E] = place;
    if (out.tiles) {
      for (uint32_t j = 0; j < tiles; j++)
        out.tiles[tile - tiles + j] = MoeTile{e, e, place - all + j * out.rows, min(out.rows, all - j * out.rows)};
      if (e == kMostExperts - 1) *out.n_tiles = tile;
    }
  }
}

// How many ids a work-group sorts, and how many work-groups that is.
inline uint32_t slice_of(uint32_t A) {
  const uint32_t n = (A + kSlice - 1) / kSlice;
  return kSlice * ((n + kMostSlices - 1) / kMostSlices);
}
inline uint32_t slices_of(uint32_t A) { return A ? (A + slice_of(A) - 1) / slice_of(A) : 0; }

}  // namespace c0ven
