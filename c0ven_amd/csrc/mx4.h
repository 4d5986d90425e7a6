// Microscaled 4-bit floats (MX4) on the device: the rows' layout, the conversions and the matrix-core product.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../../include/c0ven_quant.h"
#include "device_math.h"

namespace c0ven {

constexpr uint32_t kMxBlock = 32;  // values under one scale
constexpr uint32_t kMxRow = 128;   // a row's padding: one 16x16x128 or two 32x32x64 matrix instructions' k

__host__ __device__ constexpr uint32_t mx_steps(uint32_t cols) { return (cols + kMxRow - 1) / kMxRow; }

typedef int mx_i4 __attribute__((ext_vector_type(4)));
typedef int mx_i8 __attribute__((ext_vector_type(8)));
typedef float mx_f2 __attribute__((ext_vector_type(2)));
typedef float mx_f4 __attribute__((ext_vector_type(4)));
typedef float mx_f16 __attribute__((ext_vector_type(16)));

// The element types of operator buffers as template arguments.
template <uint32_t kType>
struct Elem;
template <>
struct Elem<QT_F32> {
  typedef float T;
};
template <>
struct Elem<QT_F16> {
  typedef _Float16 T;
};
template <>
struct Elem<QT_BF16> {
  typedef __bf16 T;
};

// A block's scale byte from the bits of its largest |x| (a float without its sign): 2^(floor(log2 m) - 2), at least
// 2^-127, in the exponent's own bias; 255 for an infinity or a NaN, whose bits are the largest. (Exponent field 0, the
// subnormal floats, is below 2^-126: also 2^-127.)
__device__ __forceinline__ uint32_t mx_scale_of(uint32_t most) {
  const uint32_t e = most >> 23;
  return e == 255 ? 255u : e > 2 ? e - 2 : 0u;
}
// The power of two of a scale byte as a float (255: NaN): exact, 2^-127 as a subnormal.
__device__ __forceinline__ float mx_pow2(uint32_t s) {
  return __uint_as_float(s == 255 ? 0x7fc00000u : s ? s << 23 : 0x00400000u);
}

// Eight values under scale byte s as a word of codes (value i in bits 4 i): round to nearest even, at most 6 in size.
// The conversion divides by the power of two in its scale operand's exponent field.
__device__ __forceinline__ uint32_t mx_codes8(const float v[8], uint32_t s) {
  const float scale = __uint_as_float(s << 23);
  uint32_t c = 0;
  c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[0], v[1], scale, 0);
  c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[2], v[3], scale, 1);
  c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[4], v[5], scale, 2);
  c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[6], v[7], scale, 3);
  return c;
}

// The values of a word of eight codes under a power of two (a float: mx_pow2), exactly, unless it leaves fp32's range.
__device__ __forceinline__ void mx_values8(uint32_t codes, float pow2, float v[8]) {
#pragma unroll
  for (int j = 0; j < 8; j++) {
    const uint32_t q = codes >> (4 * j) & 15, m = q & 7;
    const float a = m < 2 ? 0.5f * (float)m : __uint_as_float(((m >> 1) + 126) << 23 | (m & 1) << 22);
    v[j] = (q & 8 ? -a : a) * pow2;
  }
}

// exp(x) to about one unit of the last place: 2^(x log2 e) with the product's low part (v_exp_f32 is good to a unit; the
// product alone would lose |x| units). 0 below -104, infinite above 89; NaN stays.
__device__ __forceinline__ float exp_f32(float x) {
  x = x < -104.0f ? -104.0f : x > 89.0f ? 89.0f : x;
  const float hi = x * 1.4426950216e+0f;
  const float lo = __builtin_fmaf(x, 1.9259629911e-8f, __builtin_fmaf(x, 1.4426950216e+0f, -hi));
  return __builtin_amdgcn_exp2f(hi) * __builtin_fmaf(lo, 0.69314718f, 1.0f);
}

// Eight neighbours of a row, from column c on: one (two for fp32) 16-byte access where all eight are there, at whatever
// address (global memory takes it at any; rows of odd strides lose a little to the lines they share).
template <uint32_t kType>
__device__ __forceinline__ void load8(const typename Elem<kType>::T *row, uint32_t c, uint32_t cols, float v[8]) {
  typedef typename Elem<kType>::T T;
  struct __attribute__((packed)) Pack {
    T e[8];
  };
  if (c + 8 <= cols) {
    const Pack p = *(const Pack *)(row + c);
#pragma unroll
    for (int j = 0; j < 8; j++) v[j] = (float)p.e[j];
  } else {
#pragma unroll
    for (uint32_t j = 0; j < 8; j++) v[j] = c + j < cols ? (float)row[c + j] : 0.0f;
  }
}
template <uint32_t kType>
__device__ __forceinline__ void store8(typename Elem<kType>::T *row, uint32_t c, uint32_t cols, const float v[8]) {
  typedef typename Elem<kType>::T T;
  struct __attribute__((packed)) Pack {
    T e[8];
  };
  if (c + 8 <= cols) {
    Pack p;
#pragma unroll
    for (int j = 0; j < 8; j++) p.e[j] = (T)v[j];
    *(Pack *)(row + c) = p;
  } else {
#pragma unroll
    for (uint32_t j = 0; j < 8; j++)
      if (c + j < cols) row[c + j] = (T)v[j];
  }
}

// A block of 32 values held eight a lane by four neighbouring lanes: this lane's word of codes and the block's scale.
__device__ __forceinline__ uint32_t mx_quantize8(const float v[8], uint32_t &scale) {
  uint32_t most = 0;
#pragma unroll
  for (int j = 0; j < 8; j++) most = max(most, __float_as_uint(v[j]) & 0x7fffffffu);
  most = max(most, dpp_u32<kDppXor1>(most));
  most = max(most, dpp_u32<kDppXor2>(most));
  scale = mx_scale_of(most);
  return scale == 255 ? 0u : mx_codes8(v, scale);
}

__device__ __forceinline__ mx_i8 mx_wide(mx_i4 a) { return mx_i8{a[0], a[1], a[2], a[3], 0, 0, 0, 0}; }

// c += a b^T on 16 rows each over k = 128: lane l gives row l % 16, values 32 (l / 16) and on (16 bytes), with that
// block's scale in byte kA or kB of sa and sb; it receives c of a's rows 4 (l / 16) + i, b's row l % 16. (The layouts
// and the sums were checked against the definition in 64 bits.)
template <int kA, int kB>
__device__ __forceinline__ mx_f4 mx_mfma16(mx_i4 a, mx_i4 b, mx_f4 c, uint32_t sa, uint32_t sb) {
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(mx_wide(a), mx_wide(b), c, 4, 4, kA, (int)sa, kB, (int)sb);
}
// The same on 32 rows each over k = 64: lane l gives row l % 32, values 32 (l / 32) and on; it receives c of a's rows
// 8 (i / 4) + 4 (l / 32) + i % 4, b's row l % 32.
template <int kA, int kB>
__device__ __forceinline__ mx_f16 mx_mfma32(mx_i4 a, mx_i4 b, mx_f16 c, uint32_t sa, uint32_t sb) {
  return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(mx_wide(a), mx_wide(b), c, 4, 4, kA, (int)sa, kB, (int)sb);
}

}  // namespace c0ven
