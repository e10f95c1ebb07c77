// Which kernels a call of lora_add takes, and how it cuts K (lora.hip).
#pragma once

#include <stdint.h>

#include <algorithm>

namespace qtts {

constexpr int kLoraFusedCols = 256;  // output columns a workgroup of the one-launch kernel holds
constexpr int kLoraOneRank = 64;     // the largest rank of the one-launch kernel: its stages fill LDS

// Blocks of the rank: one of 16 entries, or of 32 each.
inline int lora_blocks(int64_t rank) { return rank <= 16 ? 1 : (int)((rank + 31) / 32); }

// Workgroups along the rows without a plan: m, one a row, most of which lead no group and end at once, but hold a
// compute unit's LDS until they have read the index (64 rows of one adapter through gate_up, rank 16: 11.0 us); or
// fewer than m, one a group, each of which walks the slots before its own, 90 ns each (that case: 5.5 us).
inline int64_t lora_groups(int64_t m, int64_t slots) {
  const int64_t most = std::min<int64_t>(m, slots + 1) + m / 16;
  return m <= 64 && 8 * slots <= m ? most : m;
}

// Columns of a workgroup of the second product: a wave that takes 256 of a group's columns makes its t operand once for all of
// them, but the GPU wants some 4096 waves.
inline int lora_up_cols(int64_t m, int64_t n) {
  const int64_t waves = (m + 15) / 16 * ((n + 63) / 64);  // at 64 columns a wave
  return waves >= 16384 || m <= 64 ? 256 : waves >= 8192 ? 128 : 64;
}

// One launch, the first product recomputed by each workgroup along the columns, while its workgroups (two a compute unit to
// rank 16, else one) and the A blocks that they all read stay few.  Captured calls over three adapters' worth of memory, us,
// one launch / two: rank 16, o_proj of 1 row 4.9 / 7.3, gate_up of 8 rows of 8 adapters (384 workgroups, 24 MB) 7.7 / 8.4, of
// 16 of 16 (768, 48 MB) 11.1 / 9.1; rank 32, qkv of 16 of 16 (256, 32 MB) 9.9 / 11.3, of 32 of 32 (64 MB) 17.5 / 12.5; rank 64,
// gate_up of 4 of 4 (192, 48 MB) 9.7 / 10.9, of 8 of 8 (96 MB) 17.0 / 14.2; rank 8, gate_up of 16 of 16 (768, 24 MB)
// 10.7 / 8.9.  Called one by one, the second launch costs 3 us of host time more.
inline bool lora_one_launch(bool plan, int64_t m, int64_t k, int64_t rank, int64_t slots, int64_t chunks) {
  const int64_t workgroups = chunks * std::min(m, std::min(m, slots) + m / 16);
  return !plan && rank <= kLoraOneRank && workgroups <= 640 && workgroups * rank * k * 2 <= (40ll << 20);
}

}  // namespace qtts
