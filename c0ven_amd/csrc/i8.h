// 8-bit integers with a scale a row (I8) on the device: the conversions and the matrix-core products.
#pragma once

#include "mx4.h"

namespace c0ven {

constexpr uint32_t kI8Row = 128;  // a row's padding in bytes: four 32x32x32 or two 16x16x64 matrix instructions' k
__host__ __device__ constexpr uint32_t i8_steps(uint32_t cols) { return (cols + kI8Row - 1) / kI8Row; }
__host__ __device__ constexpr uint32_t i8_pitch(uint32_t cols) { return i8_steps(cols) * kI8Row; }

typedef int i8_i16 __attribute__((ext_vector_type(16)));

// A row's scale from the bits of its largest |x| (a float without its sign): that over 127, correctly rounded, at least 2^-100
// (below, the exact test of a code's border would leave fp32's range); NaN for an infinity or a NaN, whose bits are the largest.
__device__ __forceinline__ float i8_scale_of(uint32_t most) {
  const float s = __uint_as_float(most) / 127.0f;
  return most >= 0x7f800000u ? __uint_as_float(0x7fc00000u) : s < 0x1p-100f ? 0x1p-100f : s;
}
// The integer nearest to x / s (halves to even) exactly: floor of the product with 1 / s is off by at most one next to a whole
// number, where the test against the half between does not depend on it; the fused x - (k + 1/2) s has the sign of the exact one,
// since x is a multiple of 2^-149 and s of 2^-123.
__device__ __forceinline__ uint32_t i8_code(float x, float s, float inv) {
  const float k = __builtin_floorf(x * inv);
  const float d = __builtin_fmaf(-(k + 0.5f), s, x);
  const int i = (int)k;
  return (uint32_t)(i + (d > 0.0f ? 1 : d == 0.0f ? i & 1 : 0)) & 0xffu;
}
// Eight values as two words of codes. x / s to 2^-14 lies in the low bits of x (1 / s) + 1.5 2^23, rounded once to a whole number;
// where some lane's is that near a half (one group in 16), its eight by i8_code.
__device__ __forceinline__ uint2 i8_codes8(const float v[8], float s) {
  if (s != s) return make_uint2(0, 0);
  constexpr float kWhole = 12582912.0f;  // 1.5 2^23
  const float inv = __builtin_amdgcn_rcpf(s);
  uint32_t c[8];
  float off = 0.0f;
#pragma unroll
  for (int j = 0; j < 8; j++) {
    const float t = __builtin_fmaf(v[j], inv, kWhole);
    c[j] = __float_as_uint(t);
    off = __builtin_fmaxf(off, __builtin_fabsf(__builtin_fmaf(v[j], inv, kWhole - t)));
  }
  if (off > 0.5f - 0x1p-14f) {
#pragma unroll
    for (int j = 0; j < 8; j++) c[j] = i8_code(v[j], s, inv);
  }
  const auto four = [&](int j) {
    return __builtin_amdgcn_perm(__builtin_amdgcn_perm(c[j + 3], c[j + 2], 0x0c0c0400u), __builtin_amdgcn_perm(c[j + 1], c[j], 0x0c0c0400u),
                                 0x05040100u);
  };
  return make_uint2(four(0), four(4));
}
__device__ __forceinline__ uint32_t most_of8(const float v[8]) {
  uint32_t most = 0;
#pragma unroll
  for (int j = 0; j < 8; j++) most = max(most, __float_as_uint(v[j]) & 0x7fffffffu);
  return most;
}

// Eight neighbours of a row from column c on, as they lie in memory: one (two for fp32) 16-byte load at whatever address and no
// branch, so that several are on their way at once; past the row's end the load is of its last eight (cols >= 8), and values()
// moves them down and fills up with zeros.
template <uint32_t kType>
struct Eight {
  typedef typename Elem<kType>::T T;
  typedef uint32_t Quad __attribute__((ext_vector_type(4), aligned(2)));
  static constexpr int kQuads = sizeof(T) / 2;
  uint32_t d[4 * kQuads];
  __device__ __forceinline__ void load(const T *row, uint32_t c, uint32_t cols) {
    const Quad *from = (const Quad *)(row + min(c, cols - 8));
#pragma unroll
    for (int i = 0; i < kQuads; i++) {
      const Quad v = from[i];
#pragma unroll
      for (int j = 0; j < 4; j++) d[4 * i + j] = v[j];
    }
  }
  __device__ __forceinline__ void values(uint32_t c, uint32_t cols, float v[8]) {
    const uint32_t past = c + 8 > cols ? c + 8 - cols : 0;
    if (__any(past != 0)) {
      constexpr int n = 4 * kQuads;
#pragma unroll
      for (int by = 4; by >= 1; by /= 2) {  // (elements)
        const bool move = past & by;
#pragma unroll
        for (int i = 0; i < n; i++) {
          uint32_t to;
          if (sizeof(T) == 4) {
            to = i + by < n ? d[i + by] : 0u;
          } else if (by > 1) {
            to = i + by / 2 < n ? d[i + by / 2] : 0u;
          } else {
            to = __builtin_amdgcn_alignbit(i + 1 < n ? d[i + 1] : 0u, d[i], 16);
          }
          d[i] = move ? to : d[i];
        }
      }
#pragma unroll
      for (int i = 0; i < n; i++) d[i] = past >= 8 ? 0u : d[i];
    }
    struct Values {
      T e[8];
    };
    struct Words {
      uint32_t d[4 * kQuads];
    } w;
#pragma unroll
    for (int i = 0; i < 4 * kQuads; i++) w.d[i] = d[i];
    const Values e = __builtin_bit_cast(Values, w);
#pragma unroll
    for (int j = 0; j < 8; j++) v[j] = (float)e.e[j];
  }
};
// kN groups of eight, group i of rows(i) from column cols_of(i) on; rows shorter than eight element by element.
template <uint32_t kType, int kN, typename Row, typename Col>
__device__ __forceinline__ void load_eights(uint32_t cols, Row row, Col col, float v[kN][8]) {
  if (cols >= 8) {
    Eight<kType> e[kN];
#pragma unroll
    for (int i = 0; i < kN; i++) e[i].load(row(i), col(i), cols);
#pragma unroll
    for (int i = 0; i < kN; i++) e[i].values(col(i), cols, v[i]);
  } else {
#pragma unroll
    for (int i = 0; i < kN; i++)
#pragma unroll
      for (uint32_t j = 0; j < 8; j++) {
        const float x = (float)row(i)[min(j, cols - 1)];
        v[i][j] = col(i) + j < cols ? x : 0.0f;
      }
  }
}

// c += a b^T on 16 rows each over k = 64: lane l gives row l % 16, bytes 16 (l / 16) and on; it receives c of a's rows
// 4 (l / 16) + i, b's row l % 16.
__device__ __forceinline__ mx_i4 i8_mfma16(mx_i4 a, mx_i4 b, mx_i4 c) {
  return __builtin_amdgcn_mfma_i32_16x16x64_i8(a, b, c, 0, 0, 0);
}
// The same on 32 rows each over k = 32: lane l gives row l % 32, bytes 16 (l / 32) and on; it receives c of a's rows
// 8 (i / 4) + 4 (l / 32) + i % 4, b's row l % 32.
__device__ __forceinline__ i8_i16 i8_mfma32(mx_i4 a, mx_i4 b, i8_i16 c) {
  return __builtin_amdgcn_mfma_i32_32x32x32_i8(a, b, c, 0, 0, 0);
}

// A sum of codes' products as a value: the smaller scale first, so that what is between leaves fp32's range only where the value
// does (a quantised row's scale is at least 2^-100, a sum at most 2^30; of a smaller scale from elsewhere the first product may be a
// denormal number, rounded as one). A scale that is NaN stays: scales are not negative, so that their bits are ordered as they
// are, with NaN above all.
__device__ __forceinline__ float i8_value(int sum, float sx, float sw) {
  const uint32_t a = __float_as_uint(sx), b = __float_as_uint(sw);
  return (float)sum * __uint_as_float(min(a, b)) * __uint_as_float(max(a, b));
}

}  // namespace c0ven
