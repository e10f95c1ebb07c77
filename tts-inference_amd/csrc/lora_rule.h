// Which kernels a call of lora_add takes, and how it cuts K (lora.hip).
#pragma once

#include <stdint.h>

#include <algorithm>

namespace qtts {

constexpr int kLoraFusedCols = 256;  // output columns a workgroup of the one-launch kernel holds
constexpr int kLoraOneRank = 64;     // the largest rank of the one-launch kernel: its stages fill LDS

// Blocks of the rank: one of 16 entries, or of 32 each.
inline int lora_blocks(int64_t rank) { return rank <= 16 ? 1 : (int)((rank + 31) / 32); }

// Columns of a workgroup of the second product: a wave that takes 256 of a group's columns makes its t operand once for all of
// them, but the GPU wants some 4096 waves.
inline int lora_up_cols(int64_t m, int64_t n) {
  const int64_t waves = (m + 15) / 16 * ((n + 63) / 64);  // at 64 columns a wave
  return waves >= 16384 || m <= 64 ? 256 : waves >= 8192 ? 128 : 64;
}

// One launch, the first product recomputed by each workgroup along the columns: without a plan, while the A blocks that
// they all read (one a partition column block and adapter) stay under 48 MB.
inline bool lora_one_launch(bool plan, int64_t m, int64_t k, int64_t rank, int64_t slots, int64_t chunks) {
  const int64_t groups = std::min(m, slots + m / 16);
  return !plan && rank <= kLoraOneRank && chunks * groups * rank * k * 2 <= (48ll << 20);
}

}  // namespace qtts
