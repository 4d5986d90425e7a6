// Host functions that the MX4 operators share.
#pragma once

#include "mx4.h"
#include "ops.h"

#include <type_traits>

namespace c0ven {

constexpr uint32_t kMxMostRows = 1u << 27, kMxMostCols = 1u << 20;
inline bool mx4_sizes(const moe_mx4_matrix &m) { return m.cols >= 1 && m.cols <= kMxMostCols && m.rows <= kMxMostRows; }
inline void op_mx4(const moe_mx4_matrix *m) {
  op_require(m && ((m->codes && m->scales) || !m->rows), "null argument");
  op_require(op_aligned(m->codes, 16) && op_aligned(m->scales, 16), "an MX4 matrix must be 16-byte aligned");
  op_require(mx4_sizes(*m), "an MX4 matrix has 1..2^20 cols and at most 2^27 rows");
}
inline void op_work(const void *work, uint64_t bytes, uint64_t needed) {
  op_require(bytes >= needed && (work || !needed), "the work buffer is smaller than the call's work bytes");
  op_require(op_aligned(work, 16), "the work buffer must be 16-byte aligned");
}

// f with the element type as a constant.
template <typename F>
void op_by_type(uint32_t type, F f) {
  if (type == QT_F32) f(std::integral_constant<uint32_t, QT_F32>());
  if (type == QT_F16) f(std::integral_constant<uint32_t, QT_F16>());
  if (type == QT_BF16) f(std::integral_constant<uint32_t, QT_BF16>());
}

// x (m.rows rows) into m, on the current device.
void mx4_quantize_launch(uint32_t type, const void *x, uint64_t stride, const moe_mx4_matrix &m, void *stream);

}  // namespace c0ven
