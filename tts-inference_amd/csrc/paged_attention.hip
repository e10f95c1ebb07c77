// Which kernels run a paged attention call, and how its work is cut.
#include "paged_attn.h"

int qtts_launch_paged_small(const qtts::PagedLaunch& p, int dtype, hipStream_t st);
int qtts_launch_paged_many(const qtts::PagedLaunch& p, int dtype, hipStream_t st);

namespace qtts {

// Workgroups that a call's keys are cut for, where its runs of rows alone are fewer.
constexpr int kSmallGroups = 1024, kManyGroups = 512;
constexpr int kSmallRows = 16, kManyRows = 128;  // rows of a run
constexpr int kSmallLeast = 8, kManyLeast = 8;   // tiles a split

static int64_t slot_floats(int64_t rows, int64_t d) { return (rows * (d + 2) + 63) & ~63ll; }

}  // namespace qtts

int64_t qtts_paged_attention_ws_bytes(int64_t d) {
  using namespace qtts;
  const int64_t small = split_slots(kSmallGroups) * slot_floats(kSmallRows, d);
  const int64_t many = split_slots(kManyGroups) * slot_floats(kManyRows, d);
  return kCounterBytes + (small > many ? small : many) * 4;
}

int qtts_launch_paged_attention(const qtts::PagedAttentionArgs& a, int min_new, int dtype, void* ws, hipStream_t st) {
  using namespace qtts;
  const int64_t group = a.heads / a.cache.kv_heads;
  PagedLaunch p = {};
  p.a = a;
  p.counters = (unsigned*)ws;
  p.parts = (float*)((uint8_t*)ws + kCounterBytes);
  p.fill = a.rows < 256 * 16 ? (a.rows + 15) / 16 : 256;
  const bool many = a.max_new * group > kSmallRows;
  if (!many || min_new * group <= kSmallRows) {
    p.groups = kSmallGroups / a.cache.kv_heads;
    p.least = kSmallLeast;
    p.min_rows = 0;
    p.max_rows = kSmallRows;
    p.items = a.requests + p.groups;
    const int64_t rows = a.max_new * group;
    p.slot_floats = slot_floats(rows < kSmallRows ? rows : kSmallRows, a.cache.d);
    const int st_small = qtts_launch_paged_small(p, dtype, st);
    if (!many || st_small != QTTS_OK) return st_small;
    p.min_rows = kSmallRows;
    p.fill = 0;
  }
  p.groups = kManyGroups / a.cache.kv_heads;
  p.least = kManyLeast;
  p.max_rows = INT32_MAX;
  p.items = (int32_t)((a.rows * group + kManyRows - 1) / kManyRows + a.requests + p.groups);
  p.slot_floats = slot_floats(kManyRows, a.cache.d);
  return qtts_launch_paged_many(p, dtype, st);
}
