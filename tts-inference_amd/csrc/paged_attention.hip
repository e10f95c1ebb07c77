// Attention of a step's new tokens over a paged key-value cache: the plain kernel, one wave a row and head.
#include "common.h"
#include "paged_attn.h"

namespace qtts {

namespace {

template <typename T> __device__ __forceinline__ float at(const void* p, int64_t i) { return to_f32(((const T*)p)[i]); }

// Lane l has the scores of key l of each 64, then dimensions l, l + 64, ... of the result.
template <typename T> __global__ __launch_bounds__(64) void paged_attention_kernel(PagedAttentionArgs a) {
  const int row = blockIdx.x, head = blockIdx.y, lane = threadIdx.x, d = a.cache.d;
  const int kvh = head / (a.heads / a.cache.kv_heads);
  T* out = (T*)a.out + (int64_t)row * a.ldo + (int64_t)head * d;
  float m = -INFINITY, l = 0.0f, o[kPagedMaxDim / 64] = {};
  int r = 0;
  while (r < a.requests && !(a.starts[r] <= row && row < a.starts[r] + a.counts[r])) ++r;
  if (r < a.requests && a.slots[row] >= 0) {
    const int position = a.lengths[r] - a.counts[r] + row - a.starts[r];
    const T* q = (const T*)a.q + (int64_t)row * a.ldq + (int64_t)head * d;
    for (int lo = 0; lo <= position; lo += 64) {
      const int key = lo + lane;
      const bool seen = key <= position && (!a.window || key > position - a.window || key < a.sinks);
      const int shift = a.cache.page_shift;
      int64_t base = 0;
      float s = -INFINITY;
      if (seen) {
        const int64_t page = a.table[(int64_t)r * a.cols + (key >> shift)];
        base = ((page * a.cache.kv_heads + kvh) * d) << shift;
        float sum = 0.0f;
        for (int i = 0; i < d; ++i) sum += at<T>(q, i) * at<T>(a.cache.k, base + (int64_t)(key & ((1 << shift) - 1)) * d + i);
        s = sum * a.scale;
      }
      const float top = fmaxf(m, wave_max(s));
      if (top == -INFINITY) continue;
      const float p = seen ? exp2f(s - top) : 0.0f, keep = exp2f(m - top);
      l = l * keep + wave_sum(p);
      m = top;
      for (int c = 0; c < kPagedMaxDim / 64; ++c) o[c] *= keep;
      for (int j = 0; j < 64; ++j) {
        if (!__shfl((int)seen, j, 64)) continue;
        const float pj = __shfl(p, j, 64);
        const int64_t bj = ((int64_t)__shfl((int)(base >> 32), j, 64) << 32) | (uint32_t)__shfl((int)base, j, 64);
        const int off = (lo + j) & ((1 << shift) - 1);
        for (int c = 0; c < kPagedMaxDim / 64; ++c) {
          const int i = lane + 64 * c;
          if (i < d) o[c] += pj * at<T>(a.cache.v, bj + ((int64_t)i << shift) + off);
        }
      }
    }
  }
  for (int c = 0; c < kPagedMaxDim / 64; ++c) {
    const int i = lane + 64 * c;
    if (i < d) out[i] = from_f32<T>(l > 0.0f ? o[c] / l : l);
  }
}

}  // namespace

}  // namespace qtts

int qtts_launch_paged_small(const qtts::PagedLaunch& p, int dtype, hipStream_t st);

namespace qtts {

constexpr int kSmallGroups = 1024;  // workgroups that the keys of few rows are cut for
constexpr int kSmallRows = 16;

static int64_t small_slot_floats(int rows, int d) { return ((int64_t)rows * (d + 2) + 63) & ~63ll; }

}  // namespace qtts

int64_t qtts_paged_attention_ws_bytes(int64_t d) {
  using namespace qtts;
  return kCounterBytes + 2 * kSmallGroups * small_slot_floats(kSmallRows, (int)d) * 4;
}

int qtts_launch_paged_attention(const qtts::PagedAttentionArgs& a, int min_new, int dtype, void* ws, hipStream_t st) {
  using namespace qtts;
  const int64_t group = a.heads / a.cache.kv_heads;
  if (a.max_new * group <= kSmallRows) {
    PagedLaunch p = {};
    p.a = a;
    p.groups = kSmallGroups / a.cache.kv_heads;
    p.least = 8;
    p.max_rows = kSmallRows;
    p.items = a.requests + p.groups;
    p.fill = a.rows < 256 * 16 ? (a.rows + 15) / 16 : 256;
    p.counters = (unsigned*)ws;
    p.parts = (float*)((uint8_t*)ws + kCounterBytes);
    p.slot_floats = small_slot_floats((int)(a.max_new * group), a.cache.d);
    return qtts_launch_paged_small(p, dtype, st);
  }
  const dim3 grid(a.rows, a.heads);
  if (dtype == QTTS_BF16) launch(paged_attention_kernel<bf16_t>, grid, dim3(64), 0u, st, a);
  else launch(paged_attention_kernel<f16_t>, grid, dim3(64), 0u, st, a);
  return qtts_check_launch("paged_attention");
}
