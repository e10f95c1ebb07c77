// Which kernel a call of rms_norm_quant or silu_mul_quant takes (quant_rows.hip).
#pragma once

#include <stdint.h>

namespace qtts {

// The row in registers of `threads` threads, `vectors` times eight elements each; threads == 0: the row read twice.
struct RowForm { int threads, vectors; };

// Rows of up to 16384 columns stay in registers: the fewest threads, 64 to 256, that hold the row in eight elements each, then two
// to four times eight, then 512 of three or four times eight.  One workgroup a row, so up to 2^22 rows (the grid's threads stay
// within 2^31).  Beyond either the row is read twice, element by element (one norm row of 16392 columns 45 us, of 16384 3.0; 4096 rows 212
// and 36).
inline RowForm row_form(int64_t m, int64_t k) {
  const int64_t nv = (k + 7) / 8;
  if (k <= 0 || nv > 2048 || m > (1 << 22)) return {0, 0};
  if (nv <= 64) return {64, 1};
  if (nv <= 128) return {128, 1};
  const int threads = nv <= 1024 ? 256 : 512;
  return {threads, (int)((nv + threads - 1) / threads)};
}

}  // namespace qtts
