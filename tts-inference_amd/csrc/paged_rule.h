// Which keys a row of paged attention sees, and how the work is cut: plain arithmetic, shared by the kernels, their
// launchers and the CPU tests.
#pragma once

#include <stdint.h>

#ifdef __HIPCC__
#define QTTS_RULE __host__ __device__ inline
#else
#define QTTS_RULE inline
#endif

namespace qtts {

// ---- one request's rows ---------------------------------------------------------------------------

// A request as its step left it; anything that no step makes (rows outside the batch, more rows than tokens, tokens past
// the table, more rows than the call's bound) runs as a request of no rows.
struct PagedRequest {
  int32_t start, count, length;
};
QTTS_RULE PagedRequest paged_request(int32_t start, int32_t count, int32_t length, int32_t rows, int64_t capacity,
                                     int32_t max_new) {
  const bool sound = start >= 0 && count > 0 && count <= max_new && count <= length && length <= capacity &&
                     (int64_t)start + count <= rows;
  return sound ? PagedRequest{start, count, length} : PagedRequest{0, 0, 0};
}

QTTS_RULE uint32_t paged_page(int32_t page, int32_t pages) {
  return (uint32_t)page < (uint32_t)pages ? (uint32_t)page : (uint32_t)pages - 1;
}

// ---- the keys of a run of rows, as tiles of T keys ---------------------------------------------------

// Rows at positions lo..hi see keys from: the first `sinks` and those from lo - window + 1 on (no window: all), up to hi.
// As tiles of T keys: `head` of them from key 0, then those from `first` on; `count` in all.
struct KeyTiles {
  int32_t head, first, count;
};
template <int T> QTTS_RULE KeyTiles key_tiles(int32_t lo, int32_t hi, int32_t window, int32_t sinks) {
  const int32_t end = hi / T + 1;
  const int32_t low = window ? lo - window + 1 : 0;
  if (low <= 0) return {0, 0, end};
  const int32_t first = low / T, kept = sinks < low ? sinks : low;
  const int32_t reach = (kept + T - 1) / T, head = reach < first ? reach : first;
  return {head, first, head + end - first};
}
QTTS_RULE int32_t key_tile(const KeyTiles& t, int32_t i) { return i < t.head ? i : t.first + i - t.head; }

// At most so many tiles for `span` rows that follow each other, the last one at the request's last token.
template <int T> QTTS_RULE int32_t most_tiles(int32_t length, int32_t span, int32_t window, int32_t sinks) {
  const int64_t all = ((int64_t)length + T - 1) / T;
  if (!window) return (int32_t)all;
  const int64_t some = ((int64_t)(sinks < length ? sinks : length) + T - 1) / T + ((int64_t)span + window - 2) / T + 2;
  return (int32_t)(some < all ? some : all);
}

// ---- splits of the keys over workgroups -----------------------------------------------------------------

// How the tiles of a call are cut, by its runs of rows times key-value heads (`pairs`): so many workgroups in all are
// wanted, none with fewer tiles than `least`.
struct PagedCut {
  int32_t groups, least;
};
constexpr int32_t kCutGroups = 4096;  // at most

// Runs of up to 16 rows (tiles of 32 keys, four waves a workgroup, three workgroups a compute unit).  Few pairs: one round
// of workgroups, two a unit (lengths of 4 x 16000, 16 x 4000 and 1 x 65536 tokens: 44.6, 29.2 and 47.2 us captured;
// 1024 workgroups: 54.4, 36.8 and 50.8).  A workgroup's start costs about what 8 tiles do and a join as much again, so
// that 8 are the least while compute units are idle (1 x 1000: 11.3, with 16: 14.6) and 16 where half of them are busy
// (27 windows of 512: 15.3, with 8: 17.5).  Many pairs: pieces small enough to even out ragged lengths (64 x up to 8192: 221,
// in 1024 workgroups 246).
constexpr QTTS_RULE PagedCut small_cut(int64_t pairs) {
  return pairs < 128 ? PagedCut{512, 8} : pairs < 256 ? PagedCut{512, 16} : PagedCut{kCutGroups, 16};
}
// Runs of up to 128 rows (tiles of 64 keys, two workgroups a compute unit): one round of them (512 rows behind 30000 tokens:
// 176 us captured, in 256 workgroups 204, in 1024 210; 4 x 1003 behind 2500: 136, 136, 149), and whole runs sooner where each
// unit has one (8 x 300 behind 1000 under a window of 512: 31.1, with 8 tiles as the least 33.3; 1 x 1000: 24.7, with 16: 32.0).
constexpr QTTS_RULE PagedCut many_cut(int64_t pairs) { return PagedCut{512, pairs < 256 ? 8 : 16}; }

// Tiles a split, where `total` tiles (of all runs, one head) are wanted in about `groups` workgroups a head.
QTTS_RULE uint32_t tiles_a_split(uint64_t total, int32_t groups, int32_t least) {
  const uint64_t most = 0x40000000, wide = total + (uint32_t)groups - 1;
  // (a division of 64 bits is a long way on the GPU, and no total of an ordinary call needs one)
  const uint64_t c = wide >> 32 ? wide / (uint32_t)groups : (uint32_t)wide / (uint32_t)groups;
  return c < (uint64_t)least ? (uint32_t)least : (uint32_t)(c > most ? most : c);
}
// Splits of a run of up to `tiles` tiles, equal ones: tiles / share rounded to the nearest, so that a run a little longer
// than a share stays whole.
QTTS_RULE int32_t splits_of(int32_t tiles, uint32_t share) {
  const int32_t n = (int32_t)((2 * (uint32_t)tiles + share) / (2 * share));  // tiles < 2^27, share <= 2^30
  return n > 1 ? n : 1;
}
// The share of a run whose parts cost the one workgroup that joins them `part` tiles' time each: the time, share + part
// tiles / share, is least at a share of sqrt(part tiles).
// Up to 128 rows: a part costs what a tile does, about 1 us either (100 rows behind 20000 tokens, 314 tiles: 51 us in 17
// parts, 66 in 9, 76 in 39).  Up to 16 rows: by the part's numbers (1 x 65536 tokens, 16 query heads of 128 on one: 36 us in 91
// parts, 38 in 64 or 128, 64 in 256).
constexpr float kPartCost = 1.0f / 4096;
QTTS_RULE uint32_t joined_share(int32_t tiles, uint32_t share, float part) {
#ifdef __HIP_DEVICE_COMPILE__
  const uint32_t least = (uint32_t)__builtin_amdgcn_sqrtf((float)tiles * part);  // (the precise one is a long way)
#else
  const uint32_t least = (uint32_t)__builtin_sqrtf((float)tiles * part);
#endif
  return share < least ? least : share;
}
// n > 1 splits hold n - 1/2 shares or more, so that the runs that are split have at most 4/3 groups splits between them a
// head: the results in parts that are ever held.
QTTS_RULE int64_t split_slots(int64_t groups) { return groups + groups / 3; }

}  // namespace qtts
