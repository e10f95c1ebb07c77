// Page tables, positions and cache slots of a step's new tokens, from the requests' lengths; and the pages of finished
// requests back to the free list.
//
// The mathematics: three prefix sums over the requests (rows, pages needed by those that fit), then every row finds its
// request by a binary search of the rows' ends and its page either in the table (a page that the request held before) or
// in the free list at the request's place in the pages' prefix sum.  No row depends on another one's result, so one launch
// does it all: a workgroup sums over all requests by itself and takes its share of the rows.  The lengths and the count of
// taken pages may be updated in place; the workgroup that is last to have read them writes them (a ticket).
//
// Latency bounds it: 64 requests and rows 3.6 us (one wave, an empty launch takes 2.5), 200 requests and 49152 rows 7.2 us,
// where the 0.4 MB written would take 0.1: the sums' barriers, then 8 dependent LDS reads of a search.  A workgroup a
// thousand rows, a row a thread (several rows a thread: 9.8 us), and every workgroup sums for itself: a second launch would
// cost more than the 8 KB that each reads again from the L2s.
#include "common.h"
#include "paged.h"
#include "splitk.h"

namespace qtts {

namespace {

constexpr int kStepThreads = 1024;
constexpr int kStepRows = kStepThreads;  // rows a workgroup

__device__ __forceinline__ int64_t wave_scan(int64_t v) {
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int64_t up = __shfl_up(v, o, 64);
    if ((int)(threadIdx.x & 63) >= o) v += up;
  }
  return v;
}

// Inclusive sum over the workgroup's threads; `sums` holds 16 words of LDS, free to use on return.
__device__ int64_t block_scan(int64_t v, int64_t* sums) {
  v = wave_scan(v);
  const int wave = threadIdx.x >> 6;
  if ((threadIdx.x & 63) == 63) sums[wave] = v;
  __syncthreads();
  for (int w = 0; w < wave; ++w) v += sums[w];
  __syncthreads();
  return v;
}

__device__ __forceinline__ int32_t saturate(int64_t v) { return (int32_t)(v > 0x7fffffff ? 0x7fffffff : v); }

// LDS: per request its rows' end, its length before the step, its pages before it and where its column 0 would be in the
// free list (kDenied: none of its rows is live).
constexpr int32_t kDenied = INT32_MIN;

__global__ __launch_bounds__(kStepThreads) void paged_step_kernel(PagedStepArgs a) {
  extern __shared__ int32_t lds[];
  __shared__ int64_t sums[kStepThreads / 64];
  __shared__ bool last;
  int32_t *end = lds, *length = lds + a.requests, *held = length + a.requests, *base = held + a.requests;
  const int per = (a.requests + blockDim.x - 1) / blockDim.x, first = threadIdx.x * per;
  const int stop = first + per < a.requests ? first + per : a.requests;
  const int32_t taken = *a.taken;
  const int32_t available = taken >= 0 && taken <= a.pages ? a.pages - taken : 0;
  const int64_t capacity = (int64_t)a.cols << a.page_shift;
  const int32_t round = (1 << a.page_shift) - 1;

  int64_t rows = 0;
  for (int r = first; r < stop; ++r) rows += a.added[r] > 0 ? a.added[r] : 0;
  const int64_t before = block_scan(rows, sums) - rows;
  int64_t at = before, need = 0;
  for (int r = first; r < stop; ++r) {
    const int32_t n = a.added[r] > 0 ? a.added[r] : 0, have = a.lengths[r];
    at += n;
    const bool fits = have >= 0 && (int64_t)have + n <= capacity && at <= a.rows && n <= a.max_new;
    end[r] = saturate(at);
    length[r] = have;
    held[r] = have < 0 ? 0 : (int32_t)(((int64_t)have + round) >> a.page_shift);
    const int32_t want = fits ? (int32_t)(((int64_t)have + n + round) >> a.page_shift) - held[r] : 0;
    base[r] = fits ? want : kDenied;  // until the pages' sum is known
    need += want;
  }
  const int64_t pages_before = block_scan(need, sums) - need;
  int64_t upto = pages_before, got = 0;
  for (int r = first; r < stop; ++r) {
    const int32_t want = base[r];
    if (want == kDenied) continue;
    upto += want;
    if (want == 0) {
      base[r] = 0;  // its pages are all in the table
    } else if (upto <= available) {
      got += want;
      base[r] = (int32_t)(taken + upto - want) - held[r];
    } else {
      base[r] = kDenied;
    }
  }
  const int64_t total = block_scan(got, sums);  // of the threads up to this one; its barriers make the LDS arrays readable

  for (int t = blockIdx.x * kStepRows + threadIdx.x; t < a.room && t < (int)(blockIdx.x + 1) * kStepRows; t += blockDim.x) {
    int lo = 0, hi = a.requests;  // the first request that ends past t
    while (lo < hi) {
      const int mid = (lo + hi) >> 1;
      if (end[mid] > t) hi = mid;
      else lo = mid + 1;
    }
    int32_t position = -1, slot = -1;
    if (t < a.rows && lo < a.requests && base[lo] != kDenied) {
      position = length[lo] + t - (lo ? end[lo - 1] : 0);
      const int32_t column = position >> a.page_shift;
      int32_t* entry = a.table + (int64_t)lo * a.cols + column;
      int32_t page;
      if (column < held[lo]) {
        page = *entry;
      } else {
        page = a.free_pages[base[lo] + column];
        if ((position & round) == 0) *entry = page;  // a new page has one first token, among the new ones
      }
      if (page >= 0 && page <= INT32_MAX >> a.page_shift) slot = (page << a.page_shift) + (position & round);
    }
    a.positions[t] = position;
    a.slots[t] = slot;
  }

  if (gridDim.x > 1) {  // all workgroups have read lengths and taken when the last one is here
    if (threadIdx.x == 0)
      last = __hip_atomic_fetch_add(a.ticket, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == gridDim.x - 1;
    __syncthreads();
    if (!last) return;
    if (threadIdx.x == 0) reset_counter(a.ticket);
  }
  for (int r = first; r < stop; ++r) {
    const int32_t n = base[r] == kDenied ? 0 : end[r] - (r ? end[r - 1] : 0);
    a.starts[r + 1] = end[r];
    a.counts[r] = n;
    a.lengths_out[r] = length[r] + n;
  }
  if (threadIdx.x == 0) a.starts[0] = 0;
  if (threadIdx.x == blockDim.x - 1) *a.taken_out = (int32_t)(taken + total);
}

// Latency bounds it: 64 requests of 64 pages 5.4 us captured, 2048 of 7 (16 waves, each 128 requests in turn) 34.
//
// Requests' pages back: request r's page j to free[taken - (all returned) + (returned by requests before r) + j].  One
// workgroup, a wave a request.
__global__ __launch_bounds__(kStepThreads) void paged_release_kernel(const int32_t* which, int32_t* lengths,
                                                                     const int32_t* table, int requests, int cols,
                                                                     int32_t* free_pages, int pages, int32_t* taken,
                                                                     int page_shift) {
  extern __shared__ int32_t lds[];
  __shared__ int64_t sums[kStepThreads / 64];
  __shared__ int64_t all;
  int32_t *at = lds, *count = lds + requests;
  const int per = (requests + blockDim.x - 1) / blockDim.x, first = threadIdx.x * per;
  const int stop = first + per < requests ? first + per : requests;
  const int32_t before = *taken;
  int64_t mine = 0;
  for (int r = first; r < stop; ++r) {
    const int64_t have = which[r] != 0 ? lengths[r] : 0;
    int64_t n = have > 0 ? (have + (1 << page_shift) - 1) >> page_shift : 0;
    if (n > cols) n = 0;  // no length that a step made
    count[r] = (int32_t)n;
    mine += n;
  }
  const int64_t upto = block_scan(mine, sums);
  if (threadIdx.x == blockDim.x - 1) all = upto;
  __syncthreads();
  const int64_t base = before - all;
  if (base < 0 || before > pages) return;  // more pages than were taken: no state that steps made; left as it is
  int64_t next = base + upto - mine;
  for (int r = first; r < stop; ++r) {
    at[r] = (int32_t)next;
    next += count[r];
    if (which[r] != 0) lengths[r] = 0;
  }
  if (threadIdx.x == 0) *taken = (int32_t)base;
  __syncthreads();
  const int waves = blockDim.x >> 6;
  for (int r = threadIdx.x >> 6; r < requests; r += waves)
    for (int j = threadIdx.x & 63; j < count[r]; j += 64) free_pages[at[r] + j] = table[(int64_t)r * cols + j];
}

}  // namespace

}  // namespace qtts

int qtts_launch_paged_step(const qtts::PagedStepArgs& a, hipStream_t st) {
  using namespace qtts;
  const int groups = a.room > kStepRows ? (a.room + kStepRows - 1) / kStepRows : 1;
  // one wave is enough for the prefix sums of 64 requests and as many rows; 16 waves' barriers are not
  const int most = a.room > a.requests ? a.room : a.requests;
  const int threads = most <= 64 ? 64 : most <= 256 ? 256 : kStepThreads;
  launch(paged_step_kernel, dim3(groups), dim3(threads), (uint32_t)(16 * a.requests), st, a);
  return qtts_check_launch("paged_step");
}

int qtts_launch_paged_release(const int32_t* which, int32_t* lengths, const int32_t* table, int requests, int cols,
                              int32_t* free_pages, int pages, int32_t* taken, int page_shift, hipStream_t st) {
  using namespace qtts;
  const int threads = requests <= 256 ? 256 : kStepThreads;
  launch(paged_release_kernel, dim3(1), dim3(threads), (uint32_t)(8 * requests), st, which, lengths, table, requests, cols,
         free_pages, pages, taken, page_shift);
  return qtts_check_launch("paged_release");
}
