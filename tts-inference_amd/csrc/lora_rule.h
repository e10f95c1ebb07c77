// Which kernels a call of lora_add takes, and how it cuts K (lora.hip).
#pragma once

#include <stdint.h>

#include <algorithm>

namespace qtts {

constexpr int kLoraFusedCols = 256;  // output columns a workgroup of the one-launch kernel holds
constexpr int kLoraOneRank = 64;     // the largest rank of the one-launch kernel: its stages fill LDS

// Blocks of the rank: one of 16 entries, or of 32 each.
inline int lora_blocks(int64_t rank) { return rank <= 16 ? 1 : (int)((rank + 31) / 32); }

// Workgroups along the rows without a plan: of up to 64 rows the groups of 16 rows of one slot, at most, if they are fewer (each
// workgroup then looks for its own, 0.3 us; 64 rows of 8 adapters through gate_up, rank 64: 14.7 us with one a row, 13.7), else
// one a row (64 of 64: 39.4, and 39.8 with the search).  (These and the times below: captured calls over three sets of inputs.)
inline int64_t lora_groups(int64_t m, int64_t slots) {
  return m <= 64 ? std::min<int64_t>(m, std::min<int64_t>(m, slots + 1) + m / 16) : m;
}

// 16-row tiles of A (all partitions' `tiles`; past rank 16, PACK false, two a block) that a workgroup of the first product takes:
// few, and x read more often, while each of the workgroups has a compute unit; else as many as its LDS holds.  With the
// second product, few / many: rank 16 of qkv, 300 rows of 4 adapters (70 workgroups of 1) 9.6 / 9.9 us, 2048 of 8 (411)
// 22.3 / 18.6; rank 32 of gate_up, 300 of 4 (46 of 2) 14.7 / 15.9, 2048 of 64 (386) 52.0 / 48.6; rank 32 of qkv, 300 of 64 (252)
// 16.1 / 17.4, 2048 of 8 (411) 26.3 / 27.2.
inline int lora_down_tiles(int64_t groups, int tiles, bool pack) {
  const int few = pack ? 1 : 2;
  if (groups * ((tiles + few - 1) / few) <= 256) return few;
  return pack ? std::min(tiles, 4) : tiles == 2 ? 2 : 4;
}

// Parts of K with workgroups of their own in the first product, which the second adds: two for a long K while the workgroups are
// few.  K = 6144, one / two: rank 16, 64 rows of 32 adapters 10.9 / 9.8 us, 300 of 4 11.2 / 9.5, 1003 of 32 (95 workgroups)
// 14.1 / 13.7; rank 64, 300 of 4 16.2 / 14.1.  K = 2048: rank 16, 300 of 4 through o_proj 8.3 / 7.8, 64 of 64 through qkv (192
// workgroups) 11.0 / 13.0.
constexpr int64_t kLoraSplitRows = 2048;  // 128 workgroups at the least
constexpr int kLoraSplitRank = 64;
inline int lora_max_splits(int64_t m, int64_t rank) { return m <= kLoraSplitRows && rank <= kLoraSplitRank ? 2 : 1; }
inline int lora_splits(int64_t m, int64_t k, int64_t rank, int64_t workgroups) {
  return workgroups <= 128 && k >= 2048 ? lora_max_splits(m, rank) : 1;
}

// Columns of a workgroup of the second product: a wave that takes 256 of a group's columns makes its t operand once for all of
// them, but the GPU wants some 4096 waves.
inline int lora_up_cols(int64_t m, int64_t n) {
  const int64_t waves = (m + 15) / 16 * ((n + 63) / 64);  // at 64 columns a wave
  return waves >= 16384 || m <= 64 ? 256 : waves >= 8192 ? 128 : 64;
}

// One launch, the first product recomputed by each workgroup along the columns, while the workgroups (two a compute unit to rank 16,
// else one) are little more than a round of them, and both a workgroup's A (what one compute unit then loads by itself) and all
// reads of A past the L2s are small: every group's, once a die for each partition (`reads`: the partitions' workgroups along the
// columns, at most 8 of each).  us, one launch / two: rank 16, o_proj of 1 row
// 5.1 / 7.2, qkv of 16 rows of 16 adapters (17 MB) 7.4 / 7.6, of 32 of 32 (34 MB) 10.2 / 8.5; rank 32, gate_up of 32 of 4 (13 MB)
// 7.6 / 9.2, o_proj of 32 of 32 (34 MB) 9.9 / 8.4; rank 64, qkv of 4 of 4 (17 MB) 9.4 / 9.1, of 8 of 8 (34 MB) 10.6 / 10.1,
// down_proj of 1 row (768 KiB a workgroup) 12.5 / 10.2, rank 32 (384 KiB) 8.8 / 9.4; gate_up, rank 16, of 16 of 16 (768 workgroups)
// 11.0 / 8.4, rank 32, of 8 of 8 (384) 12.1 / 8.8.  Called one by one, the second launch costs 3 us of host time more.
inline bool lora_one_launch(bool plan, int64_t m, int64_t k, int64_t rank, int64_t slots, int64_t chunks, int64_t reads) {
  const int64_t groups = std::min(m, std::min(m, slots) + m / 16), a = rank * k * 2;
  return !plan && rank <= kLoraOneRank && groups * chunks <= (rank <= 16 ? 640 : 320) && a <= 400 << 10 &&
         groups * reads * a <= 20 << 20;
}

}  // namespace qtts
