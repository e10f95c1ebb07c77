// What the paged attention kernels share: the work list that every workgroup makes for itself, the join of a run's splits
// and the rows that no request has.
#pragma once

#include "common.h"
#include "paged.h"
#include "paged_rule.h"
#include "splitk.h"

namespace qtts {

constexpr float kLowest = -3.402823466e38f;  // a reference (below) that nothing has set, as one to subtract

struct PagedLaunch {
  PagedAttentionArgs a;
  int32_t min_rows, max_rows;  // requests with more than min_rows and up to max_rows (counts times query heads a key-value head)
  int32_t items;        // workgroups a key-value head in the grid
  int32_t fill;         // workgroups behind them that write the rows without a request (0: another launch does)
  unsigned* counters;   // one a split run, zero between calls
  float* parts;         // results in parts: slot s of head h at (s * kv_heads + h) * slot_floats
  int64_t slot_floats;
};

__device__ __forceinline__ PagedRequest load_request(const PagedAttentionArgs& a, int r) {
  return paged_request(a.starts[r], a.counts[r], a.lengths[r], a.rows, (int64_t)a.cols << a.cache.page_shift, a.max_new);
}

// Inclusive sum over the lanes up to each, by DPP (no LDS round trips): within rows of 16 lanes by shifts, then each row's
// total into the rows behind it.
template <int CTRL, int ROWS> __device__ __forceinline__ uint32_t dpp_moved(uint32_t v) {
  return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, ROWS, 0xF, true);
}
__device__ __forceinline__ uint32_t wave_upto(uint32_t v) {
  v += dpp_moved<0x111, 0xF>(v);  // row_shr 1, 2, 4, 8: zeros come in
  v += dpp_moved<0x112, 0xF>(v);
  v += dpp_moved<0x114, 0xF>(v);
  v += dpp_moved<0x118, 0xF>(v);
  v += dpp_moved<0x142, 0xA>(v);  // lane 15 of rows 0 and 2 to rows 1 and 3
  v += dpp_moved<0x143, 0xC>(v);  // lane 31 to rows 2 and 3
  return v;
}
// The wave's sum of 64-bit values under 2^52: the low 26 bits' sum and the rest's.
__device__ __forceinline__ uint64_t wave_sum64(uint64_t v) {
  const uint32_t lo = __builtin_amdgcn_readlane(wave_upto((uint32_t)v & 0x3ffffff), 63);
  const uint32_t hi = __builtin_amdgcn_readlane(wave_upto((uint32_t)(v >> 26)), 63);
  return ((uint64_t)hi << 26) + lo;
}

// One workgroup's share of a head: run `run` of a request whose rows begin at `row` and whose first token's position is
// `position`, against split `split` of `splits` of its key tiles (`chunk` tiles each); `slot`: the run's first place among
// the results in parts, and its counter.
struct PagedWork {
  int32_t request, row, position, count, length;
  int32_t run, split, splits, chunk, slot;
};

// Item `item` of the list: requests in order, their runs of RUN rows (a token's query heads are rows that follow each
// other), the last run first (it has the most keys), the splits of a run.  Each wave counts for itself, a lane a share of the requests: two passes over the requests' three numbers, the
// second one from the cache.  False past the end.
template <int RUN, int T>
__device__ __forceinline__ bool paged_work(const PagedLaunch& p, int item, PagedWork& w) {
  const PagedAttentionArgs& a = p.a;
  const int lane = threadIdx.x & 63, per = (a.requests + 63) >> 6, group = a.heads / a.cache.kv_heads;
  const int span = RUN / group + 2;  // tokens that a run's rows can touch
  auto runs_of = [&](const PagedRequest& r, int32_t& tiles) -> int32_t {
    const int64_t rows = (int64_t)r.count * group;
    if (rows <= p.min_rows || rows > p.max_rows) {
      tiles = 0;
      return 0;
    }
    tiles = most_tiles<T>(r.length, r.count < span ? r.count : span, a.window, a.sinks);
    return (int32_t)((rows + RUN - 1) / RUN);
  };
  PagedRequest mine = {0, 0, 0};
  uint64_t total = 0;
  uint32_t all_runs = 0;
  for (int j = 0; j < per; ++j) {
    const int r = lane * per + j;
    if (r >= a.requests) break;
    mine = load_request(a, r);
    int32_t tiles;
    const int32_t runs = runs_of(mine, tiles);
    total += (uint64_t)runs * (uint32_t)tiles;
    all_runs += runs;
  }
  const int64_t pairs = (int64_t)__builtin_amdgcn_readlane(wave_upto(all_runs), 63) * a.cache.kv_heads;
  const PagedCut cut = RUN == 16 ? small_cut(pairs) : many_cut(pairs);
  const int32_t groups = cut.groups / a.cache.kv_heads;  // a head; 0: so many heads that nothing is cut
  const uint32_t share = groups ? tiles_a_split(wave_sum64(total), groups, cut.least) : 0;
  auto items_of = [&](const PagedRequest& r, int32_t& tiles, int32_t& splits) -> int32_t {
    const int32_t runs = runs_of(r, tiles);
    const float part = RUN == 16 ? (float)(r.count * group * a.cache.d) * kPartCost : 1.0f;
    splits = groups ? splits_of(tiles, joined_share(tiles, share, part)) : 1;
    return runs * splits;
  };
  int32_t items = 0, slots = 0;
  for (int j = 0; j < per; ++j) {
    const int r = lane * per + j;
    if (r >= a.requests) break;
    if (per > 1) mine = load_request(a, r);
    int32_t tiles, splits;
    const int32_t n = items_of(mine, tiles, splits);
    items += n;
    slots += splits > 1 ? n : 0;
  }
  const int32_t upto = wave_upto(items), slot_upto = wave_upto(slots);
  const uint64_t past = __ballot(upto > item);
  if (!past) return false;
  const int owner = __ffsll((unsigned long long)past) - 1;
  int32_t left = item - __builtin_amdgcn_readlane(upto - items, owner);
  int32_t slot = __builtin_amdgcn_readlane(slot_upto - slots, owner);
  for (int j = 0; j < per; ++j) {  // the owner's requests, every lane alike
    const int r = owner * per + j;
    PagedRequest q;
    if (per > 1) {
      q = load_request(a, r);
      q = {__builtin_amdgcn_readfirstlane(q.start), __builtin_amdgcn_readfirstlane(q.count), __builtin_amdgcn_readfirstlane(q.length)};
    } else q = {__builtin_amdgcn_readlane(mine.start, owner), __builtin_amdgcn_readlane(mine.count, owner),
              __builtin_amdgcn_readlane(mine.length, owner)};
    int32_t tiles, splits;
    const int32_t n = items_of(q, tiles, splits);
    if (left < n) {
      const int32_t order = left / splits;
      w.request = r;
      w.row = q.start;
      w.count = q.count;
      w.length = q.length;
      w.position = q.length - q.count;
      w.run = n / splits - 1 - order;
      w.split = left - order * splits;
      w.splits = splits;
      w.chunk = (tiles + splits - 1) / splits;
      w.slot = slot + order * splits;
      return true;
    }
    left -= n;
    slot += splits > 1 ? n : 0;
  }
  return false;
}

// Rows that no run writes: zeros.  Which those are goes by the requests alone, as the runs do (a slot may say otherwise: -1 where a
// table's entry is no page, or none of a request's), so that every row is written once.  Group g of p.fill takes a share of the
// rows, kFillSpan at a time, and marks in LDS what the requests cover of them.
constexpr int kFillSpan = 1024;
template <typename T> __device__ __forceinline__ void fill_rows(const PagedLaunch& p, int g) {
  __shared__ uint32_t covered[kFillSpan / 32];
  const PagedAttentionArgs& a = p.a;
  const int vecs = a.heads * a.cache.d / 8, share = (a.rows + p.fill - 1) / p.fill;
  const int end = min(a.rows, (g + 1) * share);
  const i32x4_t zero = {0, 0, 0, 0};
  for (int first = g * share; first < end; first += kFillSpan) {
    const int rows = min(kFillSpan, end - first);
    if (threadIdx.x < kFillSpan / 32) covered[threadIdx.x] = 0;
    __syncthreads();
    for (int r = threadIdx.x; r < a.requests; r += blockDim.x) {
      const PagedRequest q = load_request(a, r);
      const int stop = min(q.start + q.count - first, rows);
      for (int at = max(q.start - first, 0), next; at < stop; at = next) {
        next = min((at | 31) + 1, stop);
        atomicOr(&covered[at >> 5], (uint32_t)(((1ull << (next - at)) - 1) << (at & 31)));
      }
    }
    __syncthreads();
    for (int t = 0; t < rows; ++t) {
      if ((covered[t >> 5] >> (t & 31)) & 1) continue;
      T* out = (T*)a.out + (int64_t)(first + t) * a.ldo;
      for (int i = threadIdx.x; i < vecs; i += blockDim.x) *(i32x4_t*)(out + 8 * i) = zero;
    }
    __syncthreads();
  }
}

// Maximum over the lanes that share a column: with lane ^ 32, and with lane ^ 16 where the column's four are 16 apart.
__device__ __forceinline__ float max_32(float v) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float max_16_32(float v) {
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return max_32(fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1])));
}
__device__ __forceinline__ float sum_32(float v) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
__device__ __forceinline__ float sum_16_32(float v) {
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return sum_32(__uint_as_float(r[0]) + __uint_as_float(r[1]));
}

// Two values rounded to T, the first in the low half, by conversions that the compiler schedules: it keeps the wait that an
// exponential's reader needs (with from_f32's v_cvt_f16_f32 in inline asm right behind v_exp_f32, fp16 weights came out wrong).
template <typename T> __device__ __forceinline__ uint32_t pack2(float a, float b) {
  typedef __attribute__((ext_vector_type(2))) _Float16 f16x2_t;
  if constexpr (std::is_same<T, bf16_t>::value) return pack2_f32<T>(a, b);
  else return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2_t{a, b}), f16x2_t));
}

// 2^x, the hardware's (2^-22 relative; results below 2^-126 are zero, as is 2^-inf).
__device__ __forceinline__ float exp2_hw(float x) { return __builtin_amdgcn_exp2f(x); }

// Two values of a result in parts, published and read past the caches that other dies do not see (splitk.h).
__device__ __forceinline__ void store_pair(float* p, float a, float b) {
  store_coherent((uint64_t*)p, (uint64_t)__float_as_uint(a) | ((uint64_t)__float_as_uint(b) << 32));
}
__device__ __forceinline__ f32x2_t load_pair(const float* p) {
  return __builtin_bit_cast(f32x2_t, load_coherent((const uint64_t*)p));
}

// Weights are 2^(scale (s - r) + kAim) about a score r, the reference, that moves to a tile's largest one only where that leads by
// more than kLag powers of two: most tiles leave O as it is.  An exponent is one fma with kAim - scale r, rounded; where that is past
// kFar its steps would be the weights' own (from 2^27 on they passed every range), and r is taken off the scores
// themselves, which are near each other wherever a weight is left.
//
// fp16 holds weights from 2^-24 to 2^15 alone.  kAim uses the range above 1, and the reference moves down as well, where a tile's
// largest weight would be under 1: what falls off is 2^-25 of its tile's largest weight or less, however far that lies below the
// row's, so that a long tail keeps its share.  It stays within kDeep of the largest one so far: O stays
// under 2^117 with 2^30 keys, and as many keys in tiles below that are worth 2^-26 of the result.
constexpr float kLag = 8.0f, kFar = 1024.0f, kDeep = 56.0f;
template <typename T> constexpr float kAim = std::is_same<T, f16_t>::value ? 7.0f : 0.0f;
template <typename T> constexpr float kMost = std::is_same<T, f16_t>::value ? kDeep + kLag : kLag;  // powers of two that a key passes r by
__device__ __forceinline__ float reach_of(float s, float r, float scale) { return (s - r) * scale; }

// A column's reference, its rounded negative with kAim, and the largest reference so far.
template <typename T> struct Reference {
  float r = -INFINITY, bias = kAim<T>, peak = -INFINITY;
  bool far = false;  // some column of the wave

  // A tile's largest score: whether the reference moves to it.
  __device__ __forceinline__ bool moves(float top, float scale) const {
    const float lead = reach_of(top, r, scale);
    if constexpr (std::is_same<T, f16_t>::value) return lead > kLag || (lead < -kAim<T> && reach_of(top, peak, scale) >= -kDeep);
    else return lead > kLag;
  }
  // It does, where `now`; the factor of what was summed so far.  For whole waves.
  __device__ __forceinline__ float move(bool now, float top, float scale) {
    const float keep = now ? exp2_hw(reach_of(r, top, scale)) : 1.0f;
    r = now ? top : r;
    peak = fmaxf(peak, r);
    bias = now ? __builtin_fmaf(-top, scale, kAim<T>) : bias;
    far = __any(fabsf(bias) > kFar);
    return keep;
  }
};

// One row's sums over tiles first, first + step, ... < end again, by one wave and without the matrix cores: a value that
// the row does not see cannot reach it, where a product of tiles has 0 * NaN.  For rows whose weights are sound (l finite) and
// whose sums came out infinite or NaN.  r: their reference (scores summed in another order may pass it further: to kMost, as theirs);
// dst [d], in LDS.
template <typename T, int TILE>
__device__ __forceinline__ void row_again(const PagedAttentionArgs& a, const PagedWork& w, const KeyTiles& tiles, int first,
                                          int step, int end, int kv_head, int row, int query, int hi, float r, float* dst) {
  const int lane = threadIdx.x & 63, d = a.cache.d, shift = a.cache.page_shift, mask = (1 << shift) - 1;
  const int lo = a.window ? max(0, hi - a.window + 1) : 0;
  const int32_t* table = a.table + (int64_t)w.request * a.cols;
  const T* q = (const T*)a.q + (int64_t)row * a.ldq + (int64_t)query * d;
  float sum[kPagedMaxDim / 64] = {};
#pragma unroll 1
  for (int i = first; i < end; i += step) {
    const int key = key_tile(tiles, i) * TILE + lane;
    const bool seen = lane < TILE && key <= hi && (key >= lo || key < a.sinks);
    const int64_t page = seen ? paged_page(table[key >> shift], a.cache.pages) : 0;
    const int64_t at = (page * a.cache.kv_heads + kv_head) * ((int64_t)d << shift);
    const T* k = (const T*)a.cache.k + at + (int64_t)(key & mask) * d;
    float s = 0.0f;
    if (seen) {
#pragma unroll 1
      for (int c = 0; c < d; ++c) s += to_f32(q[c]) * to_f32(k[c]);
    }
    const float weight = seen ? exp2_hw(fminf(reach_of(s, r, a.scale), kMost<T>) + kAim<T>) : 0.0f;
    const uint64_t seen_by = __ballot(seen);
#pragma unroll 1
    for (int j = 0; j < TILE; ++j) {
      if (!((seen_by >> j) & 1)) continue;
      const float wj = __shfl(weight, j, 64);
      const int64_t pj = __shfl((int)page, j, 64);
      const T* v = (const T*)a.cache.v + (pj * a.cache.kv_heads + kv_head) * ((int64_t)d << shift) + ((key - lane + j) & mask);
#pragma unroll
      for (int c = 0; c < kPagedMaxDim / 64; ++c)
        if (lane + 64 * c < d) sum[c] += wj * to_f32(v[(int64_t)(lane + 64 * c) << shift]);
    }
  }
#pragma unroll
  for (int c = 0; c < kPagedMaxDim / 64; ++c)
    if (lane + 64 * c < d) dst[lane + 64 * c] = sum[c];
}

// Orders this wave's LDS writes before its reads, and the other way round (the wave's lanes run together).
__device__ __forceinline__ void wave_lds_fence() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}

}  // namespace qtts
