// Low-rank adapters of many requests beside one shared linear.  Row r of the activations carries its
// adapter's slot s = index[r] (outside [0, slots): none); with P output partitions of rank R each,
//   t[r, p R + i] = sum_c x[r, c] A[s, p R + i, c]                              (down)
//   out[r, j] = T(base[r, j] + scaling[s] sum_{i < ranks[s]} t[r, p(j) R + i] B[s, j, i])   (up)
// with fp32 sums and one rounding, to the output's type.  Entries past a slot's rank are never used.
#include "common.h"
#include "lora.h"

using namespace qtts;

namespace qtts {

// One wave per (row, A row).
template <typename XT> __global__ __launch_bounds__(64) void lora_down_kernel(LoraArgs g) {
  const int rows_a = g.parts.count * g.rank;
  for (int64_t r = blockIdx.y; r < g.m; r += gridDim.y) {
    const int s = g.index[r];
    if (s < 0 || s >= g.slots) continue;
    const int i = blockIdx.x;
    const XT* x = (const XT*)g.x + r * g.ldx;
    const XT* a = (const XT*)g.a + ((int64_t)s * rows_a + i) * g.k;
    float acc = 0.0f;
    for (int c = threadIdx.x; c < g.k; c += 64) acc = __builtin_fmaf(to_f32(x[c]), to_f32(a[c]), acc);
    acc = wave_sum(acc);
    if (threadIdx.x == 0) g.t[r * rows_a + i] = acc;
  }
}

// One thread per output element.
template <typename XT> __global__ __launch_bounds__(256) void lora_up_kernel(LoraArgs g) {
  const int rows_a = g.parts.count * g.rank;
  const int j = blockIdx.x * 256 + threadIdx.x;
  if (j >= g.n) return;
  int p = 0;
  while (j >= g.parts.end[p]) ++p;
  for (int64_t r = blockIdx.y; r < g.m; r += gridDim.y) {
    const int s = g.index[r];
    float v = to_f32(((const XT*)g.base)[r * g.ldb + j]);
    if (s >= 0 && s < g.slots) {
      const XT* b = (const XT*)g.b + ((int64_t)s * g.n + j) * g.rank;
      const float* t = g.t + r * rows_a + p * g.rank;
      const int live = g.ranks ? min(max(g.ranks[s], 0), g.rank) : g.rank;
      float acc = 0.0f;
      for (int i = 0; i < live; ++i) acc = __builtin_fmaf(t[i], to_f32(b[i]), acc);
      v = __builtin_fmaf(acc, g.scaling[s], v);
    }
    ((XT*)g.out)[r * g.ldo + j] = from_f32<XT>(v);
  }
}

}  // namespace qtts

int64_t qtts_lora_ws_bytes(int64_t m, int64_t rows_a) { return kCounterBytes + align256(m * rows_a * 4); }

int qtts_launch_lora_add(const LoraArgs& args, int x_dtype, void* ws, hipStream_t st) {
  LoraArgs g = args;
  g.t = (float*)((char*)ws + kCounterBytes);
  const unsigned rows = (unsigned)(g.m < 65535 ? g.m : 65535);
  const dim3 down((unsigned)(g.parts.count * g.rank), rows), up((unsigned)((g.n + 255) / 256), rows);
  if (x_dtype == QTTS_BF16) {
    qtts::launch(&lora_down_kernel<bf16_t>, down, dim3(64), 0, st, g);
    qtts::launch(&lora_up_kernel<bf16_t>, up, dim3(256), 0, st, g);
  } else {
    qtts::launch(&lora_down_kernel<f16_t>, down, dim3(64), 0, st, g);
    qtts::launch(&lora_up_kernel<f16_t>, up, dim3(256), 0, st, g);
  }
  return qtts_check_launch("lora_add");
}
