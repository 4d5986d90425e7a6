// The tile product of I8 rows on the matrix cores: y tile = x rows (BM) times w rows (BN), staged through LDS.
#pragma once

#include "i8.h"
#include "mx4_gemm.h"

namespace c0ven {

// A stage of k = 128, its eight 16-byte pieces of a row exchanged as in MxStage.
template <int BM, int BN>
struct I8Stage {
  alignas(16) uint8_t x[BM * kI8Row];
  alignas(16) uint8_t w[BN * kI8Row];
};

// kRows rows as the source of stages: row r of them is row_of(r) of the `rows` at codes (less than kNowhere bytes as far as row_of
// reaches), `steps` stages each. The waves load a kilobyte of a stage each in turn; zeros stand for rows past the last.
template <int kRows, int kWaves = 4>
struct I8Source {
  static constexpr int kLoads = kRows / 8 / kWaves;
  const uint8_t *codes;
  uint64_t bytes;
  uint32_t at[kLoads];

  template <typename F>
  __device__ __forceinline__ I8Source(const int8_t *c, uint64_t rows, uint32_t steps, F row_of)
      : codes((const uint8_t *)c), bytes(rows * steps * kI8Row) {
    const uint32_t lane = threadIdx.x & 63, wave = mx_wave();
#pragma unroll
    for (int i = 0; i < kLoads; i++)
      at[i] = row_of((wave + kWaves * i) * 8 + lane / 8) * steps * kI8Row + ((lane % 8) ^ (wave % 2 * 4 + lane / 16)) * 16;
  }
  __device__ __forceinline__ void load(uint32_t k, uint8_t *to) const {
    const uint32_t off = k * kI8Row;
    const auto from = mx_buffer(codes + off, bytes > off ? bytes - off : 0);
#pragma unroll
    for (int i = 0; i < kLoads; i++) lds_dma16(from, at[i], to + (mx_wave() + kWaves * i) * 1024);
  }
};

// A work-group's kWaves waves on a tile of BM rows of x and BN rows of w: WM of them along x's rows, the others along w's, each
// on TM runs of 32 rows of x and TN runs of 32 rows of w. kApart: a wave's runs of w lie 32 times the waves apart (gate's rows
// and up's), else they follow one another. kAcross: a lane's sums are one w row's with 16 of x's, instead of one x row's with
// 16 of w's. The operands are one step of k = 32 ahead of the matrix instructions, in registers, across the stages.
template <int TM, int TN, int WM = 2, bool kApart = false, bool kAcross = false, int kWaves = 4>
struct I8Tile {
  static constexpr int WN = kWaves / WM, BM = 32 * WM * TM, BN = 32 * WN * TN;
  typedef I8Stage<BM, BN> Stage;
  i8_i16 acc[TN][TM];
  mx_i4 a[2][TN], b[2][TM];

  static __device__ __forceinline__ uint32_t x_row() { return mx_wave() % WM * 32 * TM; }
  static __device__ __forceinline__ uint32_t w_row() { return mx_wave() / WM * 32 * (kApart ? 1 : TN); }
  static constexpr uint32_t kStep = kApart ? 32 * WN : 32;  // between a wave's runs of w

  template <int j>
  __device__ __forceinline__ void read(const Stage &s) {
    const uint32_t lane = threadIdx.x & 63, q = lane / 32, r = lane % 32;
    const uint32_t at = ((2 * j + q) ^ (r / 2 % 8)) * 16;
#pragma unroll
    for (int m = 0; m < TM; m++) b[j % 2][m] = *(const mx_i4 *)(s.x + (x_row() + r + 32 * m) * kI8Row + at);
#pragma unroll
    for (int n = 0; n < TN; n++) a[j % 2][n] = *(const mx_i4 *)(s.w + (w_row() + r + kStep * n) * kI8Row + at);
  }
  template <int j>
  __device__ __forceinline__ void multiply() {
    __builtin_amdgcn_sched_barrier(0);  // (the reads of the next step are issued first)
#pragma unroll
    for (int n = 0; n < TN; n++)
#pragma unroll
      for (int m = 0; m < TM; m++)
        acc[n][m] = kAcross ? i8_mfma32(b[j % 2][m], a[j % 2][n], acc[n][m]) : i8_mfma32(a[j % 2][n], b[j % 2][m], acc[n][m]);
    __builtin_amdgcn_sched_barrier(0);
  }
  // The matrix instructions so far stay before what follows.
  __device__ __forceinline__ void pin() {
#pragma unroll
    for (int n = 0; n < TN; n++)
#pragma unroll
      for (int m = 0; m < TM; m++) asm volatile("" : "+a"(acc[n][m]));
  }
  // Stage `now`; its step 0 is in registers. After the barrier `now` is free (load() loads what comes after `next` into it) and
  // `next` is whole. Past the last stage its first step is read all the same, and not used.
  template <typename Load>
  __device__ __forceinline__ void stage(const Stage &now, const Stage &next, Load load) {
    read<1>(now);
    multiply<0>();
    read<2>(now);
    multiply<1>();
    read<3>(now);
    multiply<2>();
    pin();
    dma_barrier();
    load();
    read<0>(next);
    multiply<3>();
    pin();
  }
  // All stages 0 .. n - 1 of a product (n > 0): load(stage, k) loads stage k's codes.
  template <typename Load>
  __device__ __forceinline__ void run(Stage &s0, Stage &s1, uint32_t n, Load load) {
#pragma unroll
    for (int i = 0; i < TN; i++)
#pragma unroll
      for (int m = 0; m < TM; m++)
#pragma unroll
        for (int j = 0; j < 16; j++) acc[i][m][j] = 0;
    load(s0, 0);
    dma_barrier();
    if (n > 1) load(s1, 1);
    read<0>(s0);
    uint32_t k = 0;
    for (; k + 1 < n; k += 2) {
      stage(s0, s1, [&] {
        if (k + 2 < n) load(s0, k + 2);
      });
      stage(s1, s0, [&] {
        if (k + 3 < n) load(s1, k + 3);
      });
    }
    if (k < n) stage(s0, s1, [] {});
  }
};

}  // namespace c0ven
