// Which kernels run a paged attention call, and how its work is cut.
#include "paged_attn.h"

int qtts_launch_paged_small(const qtts::PagedLaunch& p, int dtype, hipStream_t st);
int qtts_launch_paged_many(const qtts::PagedLaunch& p, int dtype, hipStream_t st);

namespace qtts {

constexpr int kSmallRows = 16, kManyRows = 128;  // rows of a run
constexpr int kSmallTile = 32, kManyTile = 64;

static int64_t slot_floats(int64_t rows, int64_t d) { return (rows * (d + 2) + 63) & ~63ll; }

// Items a key-value head at most, of up to `runs` runs: the splits beyond one a run are bounded by the share that each of
// them holds and by the tiles that a request of this table can have.
template <int RUN, int T> static int64_t most_items(const PagedAttentionArgs& a, int64_t runs) {
  const int64_t capacity = (int64_t)a.cols << a.cache.page_shift, span = RUN / (a.heads / a.cache.kv_heads) + 2;
  const int32_t tiles = capacity ? most_tiles<T>((int32_t)capacity, (int32_t)(a.max_new < span ? a.max_new : span), a.window, a.sinks) : 0;
  int64_t most = runs;
  for (int64_t pairs : {1, 128, 256}) {  // each of the cuts that the runs may come to
    if (pairs > runs * a.cache.kv_heads) break;
    const PagedCut cut = RUN == 16 ? small_cut(pairs) : many_cut(pairs);
    const int64_t groups = cut.groups / a.cache.kv_heads;
    if (!groups) continue;
    const int64_t by_share = runs + groups, by_tiles = runs * splits_of(tiles, cut.least), n = by_share < by_tiles ? by_share : by_tiles;
    if (n > most) most = n;
  }
  return most;
}

}  // namespace qtts

// m: rows a request and key-value head at most.
int64_t qtts_paged_attention_ws_bytes(int64_t m, int64_t d) {
  using namespace qtts;
  const int64_t small = split_slots(kCutGroups) * slot_floats(m < kSmallRows ? m : kSmallRows, d);
  const int64_t many = m > kSmallRows ? split_slots(many_cut(1).groups) * slot_floats(kManyRows, d) : 0;
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
    p.min_rows = 0;
    p.max_rows = kSmallRows;
    p.items = (int32_t)most_items<kSmallRows, kSmallTile>(a, a.requests);
    const int64_t rows = a.max_new * group;
    p.slot_floats = slot_floats(rows < kSmallRows ? rows : kSmallRows, a.cache.d);
    const int st_small = qtts_launch_paged_small(p, dtype, st);
    if (!many || st_small != QTTS_OK) return st_small;
    p.min_rows = kSmallRows;
    p.fill = 0;
  }
  p.max_rows = INT32_MAX;
  p.items = (int32_t)most_items<kManyRows, kManyTile>(a, (a.rows * group + kManyRows - 1) / kManyRows + a.requests);
  p.slot_floats = slot_floats(kManyRows, a.cache.d);
  return qtts_launch_paged_many(p, dtype, st);
}
