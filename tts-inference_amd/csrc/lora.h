// Low-rank adapters of many requests beside one linear (lora.hip): the call's arguments.
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
};

struct LoraArgs {
  const void* x;
  int64_t ldx;
  const int32_t* index;  // [m], the row's slot; outside [0, slots): no adapter
  const void* a;         // [slots, parts.count * rank, k]
  const void* b;         // [slots, n, rank]
  const int32_t* ranks;  // [slots] or null
  const float* scaling;  // [slots]
  const void* base;
  int64_t ldb;
  void* out;
  int64_t ldo;
  float* t;  // [m, parts.count * rank]
  int64_t m;
  int k, n, slots, rank;
  LoraParts parts;
};

}  // namespace qtts
