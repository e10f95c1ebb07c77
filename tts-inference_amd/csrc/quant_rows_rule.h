// Which kernel a call of rms_norm_quant or silu_mul_quant takes (quant_rows.hip).
#pragma once

#include <stdint.h>

namespace qtts {

// The row in registers of `threads` threads, `vectors` times eight elements each; threads == 0: the row read twice.
struct RowForm { int threads, vectors; };

// Rows of up to 8192 columns stay in registers: the fewest threads, 64 to 256, that hold the row in eight elements
// each, then two to four times eight.  One workgroup a row, so up to 2^22 rows (the grid's threads stay within 2^30).
inline RowForm row_form(int64_t m, int64_t k) {
  const int64_t nv = (k + 7) / 8;
  if (k <= 0 || nv > 1024 || m > (1 << 22)) return {0, 0};
  if (nv <= 64) return {64, 1};
  if (nv <= 128) return {128, 1};
  return {256, (int)((nv + 255) / 256)};
}

}  // namespace qtts
