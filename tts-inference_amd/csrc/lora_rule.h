// Which kernels a call of lora_add takes, and how it cuts K (lora.hip).
#pragma once

#include <stdint.h>

#include <algorithm>

namespace qtts {

constexpr int kLoraAtiles = 4;     // 16-row tiles of A a workgroup of the first product holds
constexpr int kLoraFusedCols = 256;  // output columns a workgroup of the one-launch kernel holds
constexpr int kLoraUpCols = 256;     // and of the second product's

constexpr int kLoraOneRank = 64;     // the largest rank of the one-launch kernel: its stages fill LDS

// Parts of K of the first product on its own: as many as give 256 workgroups when every 16 rows share an adapter
// (more adapters give more), up to 4, of 512 or more of K.
inline int lora_splits(int64_t m, int64_t rows_a, int64_t k) {
  const int64_t groups = (m + 15) / 16 * ((rows_a + 16 * kLoraAtiles - 1) / (16 * kLoraAtiles));
  return (int)std::max<int64_t>(1, std::min<int64_t>({4, k / 512, 256 / std::max<int64_t>(groups, 1)}));
}

inline int64_t lora_t_stride(int64_t rows_a) { return (rows_a + 15) / 16 * 16; }

// One launch, the first product recomputed by each workgroup along the columns: without a plan, while the A blocks that
// they all read (one a partition column block and adapter) stay under 48 MB.
inline bool lora_one_launch(bool plan, int64_t m, int64_t k, int64_t rank, int64_t slots, int64_t chunks) {
  const int64_t groups = std::min(m, slots + m / 16);
  return !plan && rank <= kLoraOneRank && chunks * groups * rank * k * 2 <= (48ll << 20);
}

}  // namespace qtts
