// The tile product of MX4 rows on the matrix cores: y tile = x rows (BM) times w rows (BN), staged through LDS.
#pragma once

#include "mx4.h"

namespace c0ven {

// A buffer of n bytes from a wave-uniform address: reads past it (from kNowhere at the latest) give zeros and fault nowhere.
constexpr uint32_t kNowhere = 0xf0000000u;
__device__ __forceinline__ __amdgpu_buffer_rsrc_t mx_buffer(const uint8_t *p, uint64_t n) {
  const uint64_t b = (uint64_t)p;
  const uint32_t hi = (uint32_t)__builtin_amdgcn_readfirstlane((uint32_t)(b >> 32));
  const uint32_t lo = (uint32_t)__builtin_amdgcn_readfirstlane((uint32_t)b);
  const uint32_t size = (uint32_t)__builtin_amdgcn_readfirstlane((uint32_t)min(n, (uint64_t)kNowhere));
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
// p ^ r / 2 % 8) so that a fragment's reads (16 rows at a time) fall on all 64 banks: 142 us of a 4096 x 8192 x 8192 product
// went to the reads alone with r % 8, 98 with r / 2 % 8.
template <int BM, int BN>
struct MxStage {
  alignas(16) uint8_t x[BM * 128];
  alignas(16) uint8_t w[BN * 128];
};
// The scales of two stages, 16 bytes a row. (A load whose neighbouring lanes do not share a line takes a clock a lane, so
// eight bytes a row and stage cost as much as the codes: 53 us of the same product.)
template <int BM, int BN>
struct MxScales {
  alignas(16) uint32_t x[BM * 4];
  alignas(16) uint32_t w[BN * 4];
};

// kRows rows as the source of stages: row r of them is row_of(r) of those at codes and scales (`rows` there are, of less than
// kNowhere bytes as far as row_of reaches), `steps` of 128 values each. The waves load a kilobyte of a stage each in turn. Zeros
// stand for rows past the last and for what is past a row's end (codes and scales of zero: products of zero).
template <int kRows, int kWaves = 4>
struct MxSource {
  static constexpr int kCodes = kRows / 8 / kWaves, kScales = (kRows + 64 * kWaves - 1) / (64 * kWaves);
  const uint8_t *codes, *scales;
  uint64_t rows;
  uint32_t at[kCodes], sat[kScales], steps;

  template <typename F>
  __device__ __forceinline__ MxSource(const uint8_t *c, const uint8_t *s, uint64_t rows, uint32_t n, F row_of)
      : codes(c), scales(s), rows(rows), steps(n) {
    const uint32_t lane = threadIdx.x & 63, wave = mx_wave();
#pragma unroll
    for (int i = 0; i < kCodes; i++)
      at[i] = row_of((wave + kWaves * i) * 8 + lane / 8) * n * 64 + ((lane % 8) ^ (wave % 2 * 4 + lane / 16)) * 16;
#pragma unroll
    for (int i = 0; i < kScales; i++) sat[i] = row_of(min((wave + kWaves * i) * 64 + lane, (uint32_t)kRows - 1)) * n * 4;
  }
  // The buffer of n bytes from byte `from` on (in scalar registers, so that a lane's offsets are the same for every stage).
  static __device__ __forceinline__ __amdgpu_buffer_rsrc_t part(const uint8_t *p, uint64_t n, uint32_t from) {
    return mx_buffer(p + from, n > from ? n - from : 0);
  }
  __device__ __forceinline__ void load(uint32_t k, uint8_t *c) const {
    const uint32_t lane = threadIdx.x & 63, wave = mx_wave();
    const auto from = part(codes, rows * steps * 64, k * 128);
    const bool in = k * 128 + ((lane % 8) ^ (wave % 2 * 4 + lane / 16)) * 16 < steps * 64;
#pragma unroll
    for (int i = 0; i < kCodes; i++) lds_dma16(from, in ? at[i] : kNowhere, c + (wave + kWaves * i) * 1024);
  }
  // The scales of stages k and k + 1 (k even).
  __device__ __forceinline__ void load_scales(uint32_t k, uint32_t *s) const {
    const uint32_t lane = threadIdx.x & 63, wave = mx_wave(), left = steps - 2 * k;
    const auto from = part(scales, rows * steps * 4, k * 8);
#pragma unroll
    for (int i = 0; i < kScales; i++) {
      if (kRows % (64 * kWaves) != 0 && (wave + kWaves * i) * 64 >= kRows) continue;
      uint32_t *to = s + (wave + kWaves * i) * 256;
      if (left >= 4) {
        if (kRows >= 64 || lane < kRows) lds_dma16(from, sat[i], to);
      } else {  // word by word (a row's address is in its lane)
        for (uint32_t j = 0; j < (kRows < 64 ? kRows : 64) / 16; j++) {
          const uint32_t row = (uint32_t)__shfl((int)sat[i], (int)(16 * j + lane / 4), 64);
          lds_dma4(from, lane % 4 < left ? row + lane % 4 * 4 : kNowhere, to + j * 64);
        }
      }
    }
  }
};

// A work-group's kWaves waves on a tile of BM rows of x and BN rows of w: WM of them along x's rows, WN along w's, each on
// TM runs of 32 rows of x and TN runs of 32 rows of w. kApart: a wave's runs of w lie 32 times the waves apart (gate's rows
// and up's), else they follow one another. kAcross: a lane's sums are one w row's with 16 of x's, instead of one x row's with
// 16 of w's. The operands are one step of k = 64 ahead of the matrix instructions, in registers, across the stages.
template <int TM, int TN, int WM = 2, bool kApart = false, bool kAcross = false, int kWaves = 4>
struct MxTile {
  static constexpr int WN = kWaves / WM, BM = 32 * WM * TM, BN = 32 * WN * TN;
  typedef MxStage<BM, BN> Stage;
  typedef MxScales<BM, BN> Scales;
  mx_f16 acc[TN][TM];
  mx_i4 a[2][TN], b[2][TM];
  uint32_t sx[TM][4], sw[TN][4];        // the pair's scales, this lane's block of each 128 in the lowest byte
  uint32_t next_sx[TM][4], next_sw[TN][4];  // the next pair's words

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

  // The next pair's scales; adopted, they are the pair's.
  __device__ __forceinline__ void read_scales(const Scales &s) {
    const uint32_t r = threadIdx.x & 31;
    const auto row = [&](const uint32_t *from, uint32_t row, uint32_t (&to)[4]) {
      const uint4 v = *(const uint4 *)(from + row * 4);
      to[0] = v.x, to[1] = v.y, to[2] = v.z, to[3] = v.w;
    };
#pragma unroll
    for (int m = 0; m < TM; m++) row(s.x, x_row() + r + 32 * m, next_sx[m]);
#pragma unroll
    for (int n = 0; n < TN; n++) row(s.w, w_row() + r + kStep * n, next_sw[n]);
  }
  __device__ __forceinline__ void adopt_scales() {
    const uint32_t q = (threadIdx.x & 63) / 32;
#pragma unroll
    for (int i = 0; i < 4; i++) {
#pragma unroll
      for (int m = 0; m < TM; m++) sx[m][i] = next_sx[m][i] >> (8 * q);
#pragma unroll
      for (int n = 0; n < TN; n++) sw[n][i] = next_sw[n][i] >> (8 * q);
    }
  }
  template <int j>
  __device__ __forceinline__ void read(const Stage &s) {
    const uint32_t lane = threadIdx.x & 63, q = lane / 32, r = lane % 32;
    const uint32_t at = ((2 * j + q) ^ (r / 2 % 8)) * 16;
#pragma unroll
    for (int m = 0; m < TM; m++) b[j % 2][m] = *(const mx_i4 *)(s.x + (x_row() + r + 32 * m) * 128 + at);
#pragma unroll
    for (int n = 0; n < TN; n++) a[j % 2][n] = *(const mx_i4 *)(s.w + (w_row() + r + kStep * n) * 128 + at);
  }
  template <int kParity, int j>
  __device__ __forceinline__ void multiply() {
    constexpr int w = 2 * kParity + j / 2;
    __builtin_amdgcn_sched_barrier(0);  // (the reads of the next step are issued first)
#pragma unroll
    for (int n = 0; n < TN; n++)
#pragma unroll
      for (int m = 0; m < TM; m++)
        acc[n][m] = kAcross ? mx_mfma32<j % 2 * 2, j % 2 * 2>(b[j % 2][m], a[j % 2][n], acc[n][m], sx[m][w], sw[n][w])
                            : mx_mfma32<j % 2 * 2, j % 2 * 2>(a[j % 2][n], b[j % 2][m], acc[n][m], sw[n][w], sx[m][w]);
    __builtin_amdgcn_sched_barrier(0);
  }
  // The matrix instructions so far stay before what follows (the compiler moves them past the barrier and the loads' blocks
  // to where their sums are used next, and keeps all their operands till then: 4096 x 8192 x 8448 183 us, 168 with this).
  __device__ __forceinline__ void pin() {
#pragma unroll
    for (int n = 0; n < TN; n++)
#pragma unroll
      for (int m = 0; m < TM; m++) asm volatile("" : "+a"(acc[n][m]));
  }
  // Stage `now`, of parity kParity; its step 0 is in registers. After the barrier `now` is free (load() loads what comes after
  // `next` into it) and `next` is whole, as are, after the second of a pair, the next pair's scales. Past the last stage its
  // first step is read all the same, and not used. The reads of the scales come before load(): after it they would wait for
  // it.
  template <int kParity, typename Load>
  __device__ __forceinline__ void stage(const Stage &now, const Stage &next, const Scales &scales, Load load) {
    read<1>(now);
    multiply<kParity, 0>();
    read<2>(now);
    multiply<kParity, 1>();
    read<3>(now);
    multiply<kParity, 2>();
    pin();
    dma_barrier();
    if (kParity == 1) read_scales(scales);
    load();
    read<0>(next);
    multiply<kParity, 3>();
    pin();
    if (kParity == 1) adopt_scales();
  }
  // The first stages of n into LDS, step 0 of the first and the first pair's scales into registers.
  template <typename Load, typename LoadScales>
  __device__ __forceinline__ void start(Stage &s0, Stage &s1, Scales &scales, uint32_t n, Load load, LoadScales load_scales) {
    load(s0, 0);
    load_scales(scales, 0);
    if (n > 1) load(s1, 1);
    dma_barrier();
    read_scales(scales);
    adopt_scales();
    read<0>(s0);
    dma_barrier();  // (every wave has its scales)
    if (n > 2) load_scales(scales, 2);
  }
  // All stages 0 .. n - 1 of a product: load(stage, k) loads stage k's codes, load_scales(scales, k) stages k's and k + 1's
  // scales (k even).
  template <typename Load, typename LoadScales>
  __device__ __forceinline__ void run(Stage &s0, Stage &s1, Scales &scales, uint32_t n, Load load, LoadScales load_scales) {
    clear();
    start(s0, s1, scales, n, load, load_scales);
    uint32_t k = 0;
    for (; k + 1 < n; k += 2) {
      stage<0>(s0, s1, scales, [&] {
        if (k + 2 < n) load(s0, k + 2);
        if (k != 0 && k + 2 < n) load_scales(scales, k + 2);
      });
      stage<1>(s1, s0, scales, [&] {
        if (k + 3 < n) load(s1, k + 3);
      });
    }
    if (k < n) stage<0>(s0, s1, scales, [] {});
  }
};

}  // namespace c0ven
