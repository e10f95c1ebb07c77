// The rows of a fused qkv projection on their way to attention: RMSNorm of the query and key heads, rotation by the rows'
// positions, queries to a contiguous tensor and keys and values into the paged cache.
//
// The mathematics, in fp32 with one rounding at the end: x <- x / sqrt(mean x^2 + eps) * w, then for i < d / 2
// (x_i, x_{i + d/2}) <- (x_i cos_i - x_{i + d/2} sin_i, x_{i + d/2} cos_i + x_i sin_i).  A group of lanes takes a head of
// a row, each lane 8 columns of either half (16-byte loads), so that a rotation's pair is in one lane and the norm's sum
// is a few lane exchanges.
#include "common.h"
#include "paged.h"

namespace qtts {

namespace {

constexpr int kThreads = 256;

template <typename T> __device__ __forceinline__ void unpack8(i32x4_t v, float (&x)[8]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    x[2 * i] = to_f32(T{(uint16_t)(uint32_t)v[i]});
    x[2 * i + 1] = to_f32(T{(uint16_t)((uint32_t)v[i] >> 16)});
  }
}

template <typename T> __device__ __forceinline__ i32x4_t pack8(const float (&x)[8]) {
  i32x4_t v;
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = (int)pack2_f32<T>(x[2 * i], x[2 * i + 1]);
  return v;
}

// L lanes a head: the least power of two with 16 L >= d.
template <typename T, int L> __global__ __launch_bounds__(kThreads) void qkv_cache_kernel(QkvCacheArgs a) {
  const int heads = a.heads + 2 * a.cache.kv_heads, d = a.cache.d, half = d / 2;
  const int64_t unit = ((int64_t)blockIdx.x * kThreads + threadIdx.x) / L;
  const int lane = threadIdx.x & (L - 1), col = lane * 8;
  const int64_t row = unit / heads;
  const int head = (int)(unit - row * heads);
  const bool live = row < a.rows;
  const bool mine = live && col < half;
  const int32_t slot = live ? a.slots[row] : -1;
  const bool kept = slot >= 0 && (slot >> a.cache.page_shift) < a.cache.pages;
  const T* src = (const T*)a.qkv + row * a.ldqkv + (int64_t)head * d;
  i32x4_t lo = {0, 0, 0, 0}, hi = {0, 0, 0, 0};
  if (mine && kept) {
    lo = *(const i32x4_t*)(src + col);
    hi = *(const i32x4_t*)(src + half + col);
  }
  const bool is_q = head < a.heads, is_v = head >= a.heads + a.cache.kv_heads;
  if (!is_v) {
    float x[8], y[8];
    unpack8<T>(lo, x);
    unpack8<T>(hi, y);
    const T* weight = (const T*)(is_q ? a.q_norm : a.k_norm);
    float sum = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) sum += x[i] * x[i] + y[i] * y[i];
#pragma unroll
    for (int o = 1; o < L; o <<= 1) sum += __shfl_xor(sum, o, 64);
    if (mine && weight) {
      const float inv = 1.0f / sqrtf(sum / (float)d + a.eps);
      float wx[8], wy[8];
      unpack8<T>(*(const i32x4_t*)(weight + col), wx);
      unpack8<T>(*(const i32x4_t*)(weight + half + col), wy);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        x[i] = x[i] * inv * wx[i];
        y[i] = y[i] * inv * wy[i];
      }
    }
    if (mine && kept && a.cos) {
      int32_t position = a.positions[row];
      position = position < 0 ? 0 : position < a.rope_rows ? position : a.rope_rows - 1;
      const float* cos = a.cos + (int64_t)position * half + col;
      const float* sin = a.sin + (int64_t)position * half + col;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float c = cos[i], s = sin[i], u = x[i], v = y[i];
        x[i] = u * c - v * s;
        y[i] = v * c + u * s;
      }
    }
    lo = pack8<T>(x);
    hi = pack8<T>(y);
  }
  if (!mine) return;
  if (is_q) {  // a row of no request: zeros
    T* q = (T*)a.q + (row * a.heads + head) * d;
    *(i32x4_t*)(q + col) = lo;
    *(i32x4_t*)(q + half + col) = hi;
    return;
  }
  if (!kept) return;
  const int kvh = head - a.heads - (is_v ? a.cache.kv_heads : 0);
  const int64_t page = slot >> a.cache.page_shift, off = slot & ((1 << a.cache.page_shift) - 1);
  const int64_t at = ((page * a.cache.kv_heads + kvh) * d) << a.cache.page_shift;
  if (!is_v) {
    T* k = (T*)a.cache.k + at + off * d;
    *(i32x4_t*)(k + col) = lo;
    *(i32x4_t*)(k + half + col) = hi;
    return;
  }
  T* v = (T*)a.cache.v + at + off;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int sh = 16 * (i & 1);
    v[(int64_t)(col + i) << a.cache.page_shift] = T{(uint16_t)((uint32_t)lo[i >> 1] >> sh)};
    v[(int64_t)(half + col + i) << a.cache.page_shift] = T{(uint16_t)((uint32_t)hi[i >> 1] >> sh)};
  }
}

template <typename T> void launch_qkv(const QkvCacheArgs& a, hipStream_t st) {
  const int64_t units = (int64_t)a.rows * (a.heads + 2 * a.cache.kv_heads);
  auto go = [&](auto lanes) {
    constexpr int L = decltype(lanes)::value;
    launch(qkv_cache_kernel<T, L>, dim3((uint32_t)((units * L + kThreads - 1) / kThreads)), dim3(kThreads), 0u, st, a);
  };
  const int need = a.cache.d / 16;
  if (need <= 1) go(std::integral_constant<int, 1>{});
  else if (need <= 2) go(std::integral_constant<int, 2>{});
  else if (need <= 4) go(std::integral_constant<int, 4>{});
  else if (need <= 8) go(std::integral_constant<int, 8>{});
  else go(std::integral_constant<int, 16>{});
}

}  // namespace

}  // namespace qtts

int qtts_launch_qkv_to_cache(const qtts::QkvCacheArgs& a, int dtype, hipStream_t st) {
  if (dtype == QTTS_BF16) qtts::launch_qkv<qtts::bf16_t>(a, st);
  else qtts::launch_qkv<qtts::f16_t>(a, st);
  return qtts_check_launch("qkv_to_cache");
}
