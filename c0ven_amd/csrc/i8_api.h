// Host functions that the I8 operators share.
#pragma once

#include "i8.h"
#include "mx4_api.h"
#include "ops.h"

namespace c0ven {

constexpr uint32_t kI8MostRows = 1u << 27, kI8MostCols = 1u << 16;
inline bool i8_sizes(const moe_i8_matrix &m) { return m.cols >= 1 && m.cols <= kI8MostCols && m.rows <= kI8MostRows; }
inline void op_i8(const moe_i8_matrix *m) {
  op_require(m && ((m->codes && m->scales) || !m->rows), "null argument");
  op_require(op_aligned(m->codes, 16) && op_aligned(m->scales, 4), "an I8 matrix's codes must be 16-byte aligned, its scales 4");
  op_require(i8_sizes(*m), "an I8 matrix has 1..65536 cols and at most 2^27 rows");
}
inline uint64_t i8_bytes(uint32_t rows, uint32_t cols) { return (uint64_t)rows * i8_pitch(cols); }

// x (m.rows rows) into m, on the current device; n_rows (device memory, or null): at most that many of them.
void i8_quantize_launch(uint32_t type, const void *x, uint64_t stride, const moe_i8_matrix &m, const uint32_t *n_rows,
                        void *stream);

}  // namespace c0ven
