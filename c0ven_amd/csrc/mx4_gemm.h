// The tile product of MX4 rows on the matrix cores: y tile = x rows (BM) times w rows (BN), staged through LDS.
#pragma once

#include "mx4.h"

namespace c0ven {

// A buffer of n bytes from a wave-uniform address: reads past it give nothing and fault nowhere.
__device__ __forceinline__ __amdgpu_buffer_rsrc_t mx_buffer(const uint8_t *p, uint64_t n) {
  const uint64_t b = (uint64_t)p;
  const uint32_t hi = (uint32_t)__builtin_amdgcn_readfirstlane((uint32_t)(b >> 32));
  const uint32_t lo = (uint32_t)__builtin_amdgcn_readfirstlane((uint32_t)b);
  const uint32_t size = (uint32_t)__builtin_amdgcn_readfirstlane((uint32_t)min(n, (uint64_t)0xffffffffu));
  return __builtin_amdgcn_make_buffer_rsrc((void *)(((uint64_t)hi << 32) | lo), 0, size, 0x00020000u);
}
// 16 (or 4) bytes a lane from off into LDS at to + 16 (4) * lane (to wave-uniform).
__device__ __forceinline__ void lds_dma16(__amdgpu_buffer_rsrc_t from, uint32_t off, void *to) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(from, (__attribute__((address_space(3))) void *)to, 16, off, 0, 0, 0);
}
__device__ __forceinline__ void lds_dma4(__amdgpu_buffer_rsrc_t from, uint32_t off, void *to) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(from, (__attribute__((address_space(3))) void *)to, 4, off, 0, 0, 0);
}
__device__ __forceinline__ uint32_t mx_wave() { return (uint32_t)__builtin_amdgcn_readfirstlane(threadIdx.x >> 6); }

// This wave's loads into LDS have arrived and its reads of LDS are done; then every wave's.
__device__ __forceinline__ void dma_barrier() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup");
  __builtin_amdgcn_s_waitcnt(0x0070);  // vmcnt(0) lgkmcnt(0)
  __builtin_amdgcn_s_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup");
}

// One stage of k = 256: 128 bytes of codes a row, its eight 16-byte pieces exchanged by the row (piece p of row r at
// p ^ r % 8) so that a fragment's reads fall on all banks; two words of scales a row.
template <int BM, int BN>
struct MxStage {
  alignas(16) uint8_t x[BM * 128];
  alignas(16) uint8_t w[BN * 128];
  alignas(16) uint32_t sx[BM * 2];
  alignas(16) uint32_t sw[BN * 2];
};

// kRows rows as the source of stages: row r of them is row_of(r) of those at codes and scales (`rows` there are), `steps`
// of 128 values each. A wave loads every fourth kilobyte of a stage. Rows past the last are out of the buffer (their results
// are not stored); what would lie past a row's end (a last stage of 128 values) is read from before it, and not used.
template <int kRows>
struct MxSource {
  static constexpr int kCodes = kRows / 32, kScales = (kRows + 127) / 128;
  __amdgpu_buffer_rsrc_t codes, scales;
  uint32_t at[kCodes], sat[kScales];

  template <typename F>
  __device__ __forceinline__ MxSource(const uint8_t *c, const uint8_t *s, uint64_t rows, uint32_t steps, F row_of)
      : codes(mx_buffer(c, rows * steps * 64)), scales(mx_buffer(s, rows * steps * 4)) {
    const uint32_t lane = threadIdx.x & 63, wave = mx_wave();
#pragma unroll
    for (int i = 0; i < kCodes; i++) at[i] = row_of((wave + 4 * i) * 8 + lane / 8) * steps * 64;
#pragma unroll
    for (int i = 0; i < kScales; i++) sat[i] = row_of(min((wave + 4 * i) * 32 + lane / 2, (uint32_t)kRows - 1)) * steps * 4;
  }
  // Stage k, from `rows` rows on.
  __device__ __forceinline__ void load(uint32_t k, uint32_t steps, uint8_t *c, uint32_t *s, uint32_t rows = 0) const {
    const uint32_t lane = threadIdx.x & 63, wave = mx_wave();
    const uint32_t col = min(k * 128 + ((lane % 8) ^ (lane / 8)) * 16, steps * 64 - 16) + rows * steps * 64;
    const uint32_t scol = min(k * 8 + lane % 2 * 4, steps * 4 - 4) + rows * steps * 4;
#pragma unroll
    for (int i = 0; i < kCodes; i++) lds_dma16(codes, at[i] + col, c + (wave + 4 * i) * 1024);
#pragma unroll
    for (int i = 0; i < kScales; i++)
      if (kRows % 128 == 0 || (wave + 4 * i) * 32 < kRows) lds_dma4(scales, sat[i] + scol, s + (wave + 4 * i) * 64);
  }
};

// A work-group's four waves on a tile of BM rows of x and BN rows of w: WM of them along x's rows, 4 / WM along w's, each on
// TM runs of 32 rows of x and TN runs of 32 rows of w. kApart: a wave's runs of w lie 32 times the waves apart (gate's rows
// and up's), else they follow one another. kAcross: a lane's sums are one w row's with 16 of x's, instead of one x row's with 16
// of w's. The operands are one step of k = 64 ahead of the matrix instructions, in
// registers, across the stages.
template <int TM, int TN, int WM = 2, bool kApart = false, bool kAcross = false>
struct MxTile {
  static constexpr int WN = 4 / WM, BM = 32 * WM * TM, BN = 32 * WN * TN;
  typedef MxStage<BM, BN> Stage;
  mx_f16 acc[TN][TM];
  mx_i4 a[2][TN], b[2][TM];
  uint32_t sx[2][TM][2], sw[2][TN][2];

  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int n = 0; n < TN; n++)
#pragma unroll
      for (int m = 0; m < TM; m++)
#pragma unroll
        for (int i = 0; i < 16; i++) acc[n][m][i] = 0.0f;
  }
  static __device__ __forceinline__ uint32_t x_row() { return mx_wave() % WM * 32 * TM; }
  static __device__ __forceinline__ uint32_t w_row() { return mx_wave() / WM * 32 * (kApart ? 1 : TN); }
  static constexpr uint32_t kStep = kApart ? 32 * WN : 32;  // between a wave's runs of w

  template <int kParity>
  __device__ __forceinline__ void read_scales(const Stage &s) {
    const uint32_t lane = threadIdx.x & 63, q = lane / 32, r = lane % 32;
#pragma unroll
    for (int m = 0; m < TM; m++) {
      const uint2 v = *(const uint2 *)(s.sx + (x_row() + r + 32 * m) * 2);
      sx[kParity][m][0] = v.x >> (8 * q), sx[kParity][m][1] = v.y >> (8 * q);
    }
#pragma unroll
    for (int n = 0; n < TN; n++) {
      const uint2 v = *(const uint2 *)(s.sw + (w_row() + r + kStep * n) * 2);
      sw[kParity][n][0] = v.x >> (8 * q), sw[kParity][n][1] = v.y >> (8 * q);
    }
  }
  template <int j>
  __device__ __forceinline__ void read(const Stage &s) {
    const uint32_t lane = threadIdx.x & 63, q = lane / 32, r = lane % 32;
    const uint32_t at = ((2 * j + q) ^ (r % 8)) * 16;
#pragma unroll
    for (int m = 0; m < TM; m++) b[j % 2][m] = *(const mx_i4 *)(s.x + (x_row() + r + 32 * m) * 128 + at);
#pragma unroll
    for (int n = 0; n < TN; n++) a[j % 2][n] = *(const mx_i4 *)(s.w + (w_row() + r + kStep * n) * 128 + at);
  }
  template <int kParity, int j>
  __device__ __forceinline__ void multiply() {
    __builtin_amdgcn_sched_barrier(0);  // (the reads of the next step are issued first)
#pragma unroll
    for (int n = 0; n < TN; n++)
#pragma unroll
      for (int m = 0; m < TM; m++)
        acc[n][m] = kAcross ? mx_mfma32<j % 2 * 2, j % 2 * 2>(b[j % 2][m], a[j % 2][n], acc[n][m], sx[kParity][m][j / 2], sw[kParity][n][j / 2])
                            : mx_mfma32<j % 2 * 2, j % 2 * 2>(a[j % 2][n], b[j % 2][m], acc[n][m], sw[kParity][n][j / 2], sx[kParity][m][j / 2]);
    __builtin_amdgcn_sched_barrier(0);
  }
  // Stage `now`, of parity kParity; its step 0 is in registers. half: the row ends after its first two steps. After the
  // barrier `now` is free (load() loads what comes after `next` into it) and `next` is whole; past the last stage its first
  // step is read all the same, and not used. (The two halves are basic blocks of their own: 64 matrix instructions on all
  // 256 accumulators in one are more than the compiler's register allocation holds without spills.)
  template <int kParity, typename Load>
  __device__ __forceinline__ void stage(const Stage &now, const Stage &next, bool half, Load load) {
    read<1>(now);
    multiply<kParity, 0>();
    read<2>(now);
    multiply<kParity, 1>();
    if (!half) {
      read<3>(now);
      multiply<kParity, 2>();
      dma_barrier();
      load();
      read<0>(next);
      read_scales<kParity ^ 1>(next);
      multiply<kParity, 3>();
    } else {
      dma_barrier();
      load();
      read<0>(next);
      read_scales<kParity ^ 1>(next);
    }
  }
  __device__ __forceinline__ void start(const Stage &first) {
    read<0>(first);
    read_scales<0>(first);
  }
};

}  // namespace c0ven
