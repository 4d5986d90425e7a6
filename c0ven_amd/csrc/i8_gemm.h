// The tile product of I8 rows on the matrix cores: y tile = x rows (BM) times w rows (BN), staged through LDS.
#pragma once

#include "i8.h"
#include "mx4_gemm.h"

namespace c0ven {

// A barrier at which all but the wave's last kLoads loads have arrived (no fence: it would wait for all).
template <int kLoads>
__device__ __forceinline__ void dma_barrier_but() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt(0x0070 | kLoads % 16 | kLoads / 16 << 14);  // vmcnt(kLoads) lgkmcnt(0)
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

// A stage of k = 128, its eight 16-byte pieces of a row exchanged as in MxStage.
template <int kRows>
struct I8Rows {
  alignas(16) uint8_t b[kRows * kI8Row];
};

// kRows rows as the source of stages: row r of them is row_of(r) of the `rows` at codes (less than kNowhere bytes as far as row_of
// reaches), `steps` stages each. The waves load a kilobyte of a stage each in turn; zeros stand for rows past the last.
template <int kRows, int kWaves = 4>
struct I8Source {
  static constexpr int kLoads = kRows / 8 / kWaves;
  const uint8_t *codes;
  uint64_t bytes;
  uint32_t at[kLoads];

  // The row of a stage that this lane's load i is of.
  static __device__ __forceinline__ uint32_t row(int i) { return (mx_wave() + kWaves * i) * 8 + (threadIdx.x & 63) / 8; }
  __device__ __forceinline__ void aim(int i, uint32_t r, uint32_t steps) {
    const uint32_t lane = threadIdx.x & 63;
    at[i] = r * steps * kI8Row + ((lane % 8) ^ (mx_wave() % 2 * 4 + lane / 16)) * 16;
  }
  __device__ __forceinline__ void move(const int8_t *c, uint64_t rows, uint32_t steps) {
    codes = (const uint8_t *)c, bytes = rows * steps * kI8Row;
  }
  template <typename F>
  __device__ __forceinline__ I8Source(const int8_t *c, uint64_t rows, uint32_t steps, F row_of) {
    move(c, rows, steps);
#pragma unroll
    for (int i = 0; i < kLoads; i++) aim(i, row_of(row(i)), steps);
  }
  // Stage k, zeros unless k < end.
  __device__ __forceinline__ void load(uint32_t k, uint8_t *to, uint32_t end = ~0u) const {
    const uint32_t off = k * kI8Row;
    const auto from = mx_buffer(codes + off, k < end && bytes > off ? bytes - off : 0);
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
  typedef I8Rows<BM> X;
  typedef I8Rows<BN> W;
  i8_i16 acc[TN][TM];
  mx_i4 a[2][TN], b[2][TM];

  static __device__ __forceinline__ uint32_t x_row() { return mx_wave() % WM * 32 * TM; }
  static __device__ __forceinline__ uint32_t w_row() { return mx_wave() / WM * 32 * (kApart ? 1 : TN); }
  static constexpr uint32_t kStep = kApart ? 32 * WN : 32;  // between a wave's runs of w

  template <int j>
  __device__ __forceinline__ void read(const X &x, const W &w) {
    const uint32_t lane = threadIdx.x & 63, q = lane / 32, r = lane % 32;
    const uint32_t at = ((2 * j + q) ^ (r / 2 % 8)) * 16;
#pragma unroll
    for (int m = 0; m < TM; m++) b[j % 2][m] = *(const mx_i4 *)(x.b + (x_row() + r + 32 * m) * kI8Row + at);
#pragma unroll
    for (int n = 0; n < TN; n++) a[j % 2][n] = *(const mx_i4 *)(w.b + (w_row() + r + kStep * n) * kI8Row + at);
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
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int n = 0; n < TN; n++)
#pragma unroll
      for (int m = 0; m < TM; m++)
#pragma unroll
        for (int j = 0; j < 16; j++) acc[n][m][j] = 0;
  }
  // Stage x, w; its step 0 is in registers. barrier() waits for the next stage's loads and for every wave; then x and w are free
  // (load() loads what comes later into them). Past the last stage its first step is read all the same, and not used.
  template <typename Barrier, typename Load>
  __device__ __forceinline__ void stage(const X &x, const W &w, const X &next_x, const W &next_w, Barrier barrier, Load load) {
    read<1>(x, w);
    multiply<0>();
    read<2>(x, w);
    multiply<1>();
    read<3>(x, w);
    multiply<2>();
    pin();
    barrier();
    load();
    read<0>(next_x, next_w);
    multiply<3>();
    pin();
  }
  // All stages 0 .. n - 1 of a product (n > 0), two buffers each: load_x(buffer, k) and load_w load stage k's codes.
  template <typename LoadX, typename LoadW>
  __device__ __forceinline__ void run2(X &x0, X &x1, W &w0, W &w1, uint32_t n, LoadX load_x, LoadW load_w) {
    clear();
    load_w(w0, 0), load_x(x0, 0);
    dma_barrier();
    if (n > 1) load_w(w1, 1), load_x(x1, 1);
    read<0>(x0, w0);
    uint32_t k = 0;
    for (; k + 1 < n; k += 2) {
      stage(x0, w0, x1, w1, dma_barrier, [&] {
        if (k + 2 < n) load_w(w0, k + 2), load_x(x0, k + 2);
      });
      stage(x1, w1, x0, w0, dma_barrier, [&] {
        if (k + 3 < n) load_w(w1, k + 3), load_x(x1, k + 3);
      });
    }
    if (k < n) stage(x0, w0, x1, w1, dma_barrier, [] {});
  }
  // Products of n stages (n even) one after another, the next one's first two loaded in the last two of this: begin() at a
  // product's first stage, turn() from where the loads are the next product's, done() when its sums are there; false ends it.
  // done()'s kStores stores (a wave's) go on beside the first stage: its barrier waits for what was loaded before them.
  template <int kStores, typename LoadX, typename LoadW, typename Begin, typename Turn, typename Done>
  __device__ __forceinline__ void run_items(X &x0, X &x1, W &w0, W &w1, uint32_t n, LoadX load_x, LoadW load_w, Begin begin, Turn turn,
                                            Done done) {
    constexpr int kBefore = kStores < 62 ? kStores : 62;  // (63 is no wait)
    const auto load0 = [&](uint32_t k) { load_w(w0, k), load_x(x0, k); };
    const auto load1 = [&](uint32_t k) { load_w(w1, k), load_x(x1, k); };
    const auto pair = [&](auto barrier, uint32_t k) {
      stage(x0, w0, x1, w1, barrier, [&] { load0(k); });
      stage(x1, w1, x0, w0, dma_barrier, [&] { load1(k + 1); });
    };
    load0(0);
    dma_barrier();
    load1(1);
    read<0>(x0, w0);
    __builtin_amdgcn_s_waitcnt(0x0f70);  // vmcnt(0) (no store is before the first)
    do {
      clear();
      begin();
      if (n == 2) turn();
      pair(dma_barrier_but<kBefore>, n == 2 ? 0 : 2);
      if (n > 2) {
        for (uint32_t k = 4; k < n; k += 2) pair(dma_barrier, k);
        turn();
        pair(dma_barrier, 0);
      }
    } while (done());
    dma_barrier_but<kBefore>();  // (LDS is another work-group's after this one)
  }
  // The same with four buffers each, so that a stage's loads have three stages' time: a barrier waits for all but the last two
  // stages' loads, kLoads a wave and stage.
  template <int kLoads, typename LoadX, typename LoadW>
  __device__ __forceinline__ void run8(X &x0, X &x1, X &x2, X &x3, W &w0, W &w1, W &w2, W &w3, uint32_t n, LoadX load_x,
                                       LoadW load_w) {
    clear();
    // (Loads without conditions, past the last stage of nothing, so that the compiler knows which are outstanding where.)
    load_w(w0, 0), load_x(x0, 0);
    load_w(w1, 1), load_x(x1, 1);
    load_w(w2, 2), load_x(x2, 2);
    load_w(w3, 3), load_x(x3, 3);
    dma_barrier_but<3 * kLoads>();
    read<0>(x0, w0);
    uint32_t k = 0;
    for (; k + 4 <= n; k += 4) {
      stage(x0, w0, x1, w1, dma_barrier_but<2 * kLoads>, [&] { load_w(w0, k + 4), load_x(x0, k + 4); });
      stage(x1, w1, x2, w2, dma_barrier_but<2 * kLoads>, [&] { load_w(w1, k + 5), load_x(x1, k + 5); });
      stage(x2, w2, x3, w3, dma_barrier_but<2 * kLoads>, [&] { load_w(w2, k + 6), load_x(x2, k + 6); });
      stage(x3, w3, x0, w0, dma_barrier_but<2 * kLoads>, [&] { load_w(w3, k + 7), load_x(x3, k + 7); });
    }
    const auto none = [] {};
    if (k < n) stage(x0, w0, x1, w1, dma_barrier_but<2 * kLoads>, none);
    if (k + 1 < n) stage(x1, w1, x2, w2, dma_barrier_but<kLoads>, none);
    if (k + 2 < n) stage(x2, w2, x3, w3, dma_barrier, none);
    dma_barrier();
  }
  // The same with three buffers of x and two of w (all of LDS with tiles of 256): x is loaded two stages ahead, so that half of a
  // stage's bytes have two stages' time, and a barrier waits for w's (and the older x's) alone: all but the last kXLoads loads of
  // a wave, which are one buffer of x's.
  template <int kXLoads, typename LoadX, typename LoadW>
  __device__ __forceinline__ void run5(X &x0, X &x1, X &x2, W &w0, W &w1, uint32_t n, LoadX load_x, LoadW load_w) {
    clear();
    load_w(w0, 0), load_x(x0, 0);
    dma_barrier();
    if (n > 1) load_x(x1, 1), load_w(w1, 1);
    if (n > 2) load_x(x2, 2);
    read<0>(x0, w0);
    uint32_t k = 0;
    const auto six = [&](auto each) {
      each(x0, w0, x1, w1, k);
      each(x1, w1, x2, w0, k + 1);
      each(x2, w0, x0, w1, k + 2);
      each(x0, w1, x1, w0, k + 3);
      each(x1, w0, x2, w1, k + 4);
      each(x2, w1, x0, w0, k + 5);
    };
    // (Without conditions, so that the compiler knows which loads are outstanding where.)
    for (; k + 8 < n; k += 6)
      six([&](X &x, W &w, const X &next_x, const W &next_w, uint32_t i) {
        stage(
            x, w, next_x, next_w,
            dma_barrier_but<kXLoads>,
            [&] { load_w(w, i + 2), load_x(x, i + 3); });
      });
    const auto last = [&](X &x, W &w, const X &next_x, const W &next_w, uint32_t i) {
      if (i < n)
        stage(x, w, next_x, next_w, dma_barrier, [&] {
          if (i + 2 < n) load_w(w, i + 2);
          if (i + 3 < n) load_x(x, i + 3);
        });
    };
    six(last);
    last(x0, w0, x1, w1, k + 6);
    last(x1, w1, x2, w0, k + 7);
  }
};

}  // namespace c0ven
