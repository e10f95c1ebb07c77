// Low-rank adapters of many requests beside one linear (lora.hip): the call's arguments and the plan's layout.
#pragma once

#include <stdint.h>

namespace qtts {

constexpr int kLoraMaxParts = 8;
constexpr int kLoraMaxRank = 128;

// Output partitions of a merged linear: partition p has columns [end[p - 1], end[p]) and rows
// [p rank, (p + 1) rank) of an adapter's A.
struct LoraParts {
  int count;
  int32_t end[kLoraMaxParts];
  int32_t chunk_end[kLoraMaxParts];  // workgroups along the columns, each within one partition
};

struct LoraArgs {
  const int32_t* index;  // [m], the row's slot; outside [0, slots): no adapter
  const int32_t* plan;   // or null
  const void* x;
  int64_t ldx;
  const void* a;         // [slots, parts.count * rank, k]
  const void* b;         // [slots, n, rank]
  const int32_t* ranks;  // [slots] or null
  const float* scaling;  // [slots]
  const void* base;
  int64_t ldb;
  void* out;
  int64_t ldo;
  uint8_t* t;     // [splits, m, parts.count, blocks]: the first product's sums as 16-bit parts (lora.hip)
  int32_t* exps;  // as many, fp16
  int64_t m;
  int k, n, slots, rank, blocks, up_cols, splits;
  int64_t groups;  // at most, of the batch: the workgroups along the rows
  bool whole;      // every row is written, by the index alone where the plan is another batch's
  LoraParts parts;
};

// ---- the plan: rows sorted by slot, cut into groups of one slot each ---------------------------
// int32 words: the number of groups, m, slots, 0; then, from word 4, two words a group (slot, or -1 for rows without an
// adapter; its rows, at most kPlanGroup); then kPlanGroup words a group, its rows.
constexpr int kPlanGroup = 16;
constexpr int kPlanMaxSlots = 768;  // the sort's counters are in LDS
constexpr int64_t kPlanMaxRows = 1 << 30;  // places in int32

__host__ __device__ inline int64_t plan_max_groups(int64_t m, int64_t slots) {
  return (m + kPlanGroup - 1) / kPlanGroup + (m < slots + 1 ? m : slots + 1);
}
__host__ __device__ inline int64_t plan_order_at(int64_t m, int64_t slots) {
  return 4 + (2 * plan_max_groups(m, slots) + 3) / 4 * 4;
}
__host__ __device__ inline int64_t plan_words(int64_t m, int64_t slots) {
  return plan_order_at(m, slots) + kPlanGroup * plan_max_groups(m, slots);
}

}  // namespace qtts
