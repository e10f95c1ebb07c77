// The rows of a fused qkv projection on their way to attention: RMSNorm of the query and key heads, rotation by the rows'
// positions, queries to a contiguous tensor and keys and values into the paged cache.
//
// The mathematics, in fp32 with one rounding at the end: x <- x / sqrt(mean x^2 + eps) * w, then for i < d / 2
// (x_i, x_{i + d/2}) <- (x_i cos_i - x_{i + d/2} sin_i, x_{i + d/2} cos_i + x_i sin_i).  A group of lanes takes a head of
// a row, each lane 8 columns of either half (16-byte loads), so that a rotation's pair is in one lane and the norm's sum
// is a few lane exchanges; workgroups of their own take the values.
//
// Memory bounds many rows: 2048 rows of 16 + 2 x 8 heads of 128 (34 MB in and out) take 9.1 us captured, 3.7 TB/s, of which
// 2.5 are an empty launch; the norm and the rotation hide behind the loads.  With values written as they come, 2 bytes a
// dimension into lines of other rows, it took 17.6.  One row is latency: 3.0 us.
#include "common.h"
#include "paged.h"

namespace qtts {

namespace {

constexpr int kThreads = 256;
// Heads of rows from which a thread takes four, which share the row's angles, and values go 64 rows a workgroup instead of 8
// (2048 rows of 16 + 8 heads: 9.3 us captured, one head and 8 rows 9.8; 512 rows 6.9 and 4.9, 64 single tokens 9.5 and 4.2).
constexpr int64_t kManyHeads = 32768;

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

// Queries and keys: L lanes a head (the least power of two with 16 L >= d), PER heads of a row one after the other.
template <typename T, int L, int PER> __device__ __forceinline__ void qk_heads(const QkvCacheArgs& a, int block) {
  const int heads = a.heads + a.cache.kv_heads, d = a.cache.d, half = d / 2, parts = (heads + PER - 1) / PER;
  const int64_t unit = ((int64_t)block * kThreads + threadIdx.x) / L;
  const int lane = threadIdx.x & (L - 1), col = lane * 8;
  const int64_t row = unit / parts;
  const int first = (int)(unit - row * parts) * PER;
  const bool live = row < a.rows, mine = live && col < half;
  const int32_t slot = live ? a.slots[row] : -1;
  const bool kept = slot >= 0 && (slot >> a.cache.page_shift) < a.cache.pages;
  const T* src = (const T*)a.qkv + row * a.ldqkv + (int64_t)first * d;
  i32x4_t lo[PER], hi[PER];
#pragma unroll
  for (int n = 0; n < PER; ++n) {
    lo[n] = hi[n] = i32x4_t{0, 0, 0, 0};
    if (mine && kept && first + n < heads) {
      lo[n] = *(const i32x4_t*)(src + n * d + col);
      hi[n] = *(const i32x4_t*)(src + n * d + half + col);
    }
  }
  float c[8], s[8];
  if (mine && kept && a.cos) {
    int32_t position = a.positions[row];
    position = position < 0 ? 0 : position < a.rope_rows ? position : a.rope_rows - 1;
#pragma unroll
    for (int i = 0; i < 8; i += 4) {
      *(f32x4_t*)(c + i) = *(const f32x4_t*)(a.cos + (int64_t)position * half + col + i);
      *(f32x4_t*)(s + i) = *(const f32x4_t*)(a.sin + (int64_t)position * half + col + i);
    }
  }
#pragma unroll
  for (int n = 0; n < PER; ++n) {
    const int head = first + n;
    const bool is_q = head < a.heads;
    float x[8], y[8];
    unpack8<T>(lo[n], x);
    unpack8<T>(hi[n], y);
    const T* weight = (const T*)(is_q ? a.q_norm : a.k_norm);
    float sum = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) sum += x[i] * x[i] + y[i] * y[i];
#pragma unroll
    for (int o = 1; o < L; o <<= 1) sum += __shfl_xor(sum, o, 64);
    if (mine && kept && weight) {  // (a norm of zeros need not be zeros)
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
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float u = x[i], v = y[i];
        x[i] = u * c[i] - v * s[i];
        y[i] = v * c[i] + u * s[i];
      }
    }
    if (!mine || head >= heads || !(is_q || kept)) continue;
    T* out;
    if (is_q) {  // a row of no request: zeros
      out = (T*)a.q + (row * a.heads + head) * d;
    } else {
      const int64_t page = slot >> a.cache.page_shift, off = slot & ((1 << a.cache.page_shift) - 1);
      out = (T*)a.cache.k + (((page * a.cache.kv_heads + head - a.heads) * d) << a.cache.page_shift) + off * d;
    }
    *(i32x4_t*)(out + col) = pack8<T>(x);
    *(i32x4_t*)(out + half + col) = pack8<T>(y);
  }
}

// Values: a workgroup takes ROWS rows of one head through LDS, since they lie d-major on their page.  Eight rows whose slots are
// eight tokens in a row from a multiple of eight go out together, 16 bytes a dimension (eight such groups fill lines of
// 128 bytes); the group belongs to the workgroup of its first row, which reads up to 7 rows past its own.  Other rows
// (a request's ends) go out by themselves, 2 bytes a dimension.
template <typename T, int ROWS> __device__ __forceinline__ void value_rows(const QkvCacheArgs& a, int tile, int h) {
  constexpr int kReach = ROWS + 8, GROUPS = ROWS / 8;
  __shared__ uint16_t rows[kReach][kPagedMaxDim + 2];
  __shared__ int32_t slot_of[kReach + 8];  // of rows first - 8 .. first + kReach - 1
  const int d = a.cache.d, wave = threadIdx.x >> 6, lane = threadIdx.x & 63, shift = a.cache.page_shift;
  const int64_t first = (int64_t)tile * ROWS;
  if (threadIdx.x < kReach + 8) {
    const int64_t row = first - 8 + threadIdx.x;
    int32_t slot = row >= 0 && row < a.rows ? a.slots[row] : -1;
    if (slot >= 0 && (slot >> shift) >= a.cache.pages) slot = -1;
    slot_of[threadIdx.x] = slot;
  }
  const uint16_t* src = (const uint16_t*)a.qkv + first * a.ldqkv + (int64_t)(a.heads + a.cache.kv_heads + h) * d;
  for (int u = threadIdx.x; u < kReach * (d / 8); u += kThreads) {
    const int r = u / (d / 8), col = (u - r * (d / 8)) * 8;
    if (first + r >= a.rows) break;
    const i32x4_t v = *(const i32x4_t*)(src + r * a.ldqkv + col);
#pragma unroll
    for (int i = 0; i < 4; ++i) *(int32_t*)&rows[r][col + 2 * i] = v[i];
  }
  __syncthreads();
  auto leads = [&](int t) {  // row first + t, t >= -7: the first of a group
    const int32_t slot = slot_of[8 + t];
    bool all = slot >= 0 && (slot & 7) == 0;
#pragma unroll
    for (int i = 1; i < 8; ++i) all = all && slot_of[8 + t + i] == slot + i;
    return all;
  };
  const int row = lane & (ROWS - 1);  // the lane's row of the tile, for the two questions asked of each
  const int32_t mine = slot_of[8 + row];
  const uint64_t leaders = __ballot(lane < ROWS && leads(row));
  uint64_t alone = __ballot(lane < ROWS && mine >= 0 && !leads(row - (mine & 7)));
  T* cache = (T*)a.cache.v;
  auto base_of = [&](int32_t slot) {
    return ((((int64_t)(slot >> shift)) * a.cache.kv_heads + h) * d << shift) + (slot & ((1 << shift) - 1));
  };
  uint64_t left = leaders;  // at most GROUPS
  for (int n = lane & (GROUPS - 1); n && left; --n) left &= left - 1;
  if (left) {
    const int t = __builtin_ctzll(left);
    T* to = cache + base_of(slot_of[8 + t]);
    for (int dim = threadIdx.x / GROUPS; dim < d; dim += kThreads / GROUPS) {
      i32x4_t v;
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = (int)(rows[t + 2 * i][dim] | ((uint32_t)rows[t + 2 * i + 1][dim] << 16));
      *(i32x4_t*)(to + ((int64_t)dim << shift)) = v;
    }
  }
  for (int n = 0; alone; ++n) {
    const int t = __builtin_ctzll(alone);
    alone &= alone - 1;
    if ((n & 3) != wave) continue;
    T* to = cache + base_of(slot_of[8 + t]);
    for (int dim = lane; dim < d; dim += 64) to[(int64_t)dim << shift] = T{rows[t][dim]};
  }
}

template <typename T, int L, int PER, int ROWS> __global__ __launch_bounds__(kThreads) void qkv_cache_kernel(QkvCacheArgs a, int value_groups) {
  if ((int)blockIdx.x < value_groups) value_rows<T, ROWS>(a, blockIdx.x / a.cache.kv_heads, blockIdx.x % a.cache.kv_heads);
  else qk_heads<T, L, PER>(a, blockIdx.x - value_groups);
}

template <typename T> void launch_qkv(const QkvCacheArgs& a, hipStream_t st) {
  const int heads = a.heads + a.cache.kv_heads;
  auto go = [&](auto lanes, auto per, auto rows) {
    constexpr int L = decltype(lanes)::value, PER = decltype(per)::value, ROWS = decltype(rows)::value;
    const int64_t values = ((int64_t)a.rows + ROWS - 1) / ROWS * a.cache.kv_heads;
    const int64_t units = (int64_t)a.rows * ((heads + PER - 1) / PER);
    launch(qkv_cache_kernel<T, L, PER, ROWS>, dim3((uint32_t)(values + (units * L + kThreads - 1) / kThreads)), dim3(kThreads), 0u, st,
           a, (int)values);
  };
  auto by_rows = [&](auto lanes) {
    if ((int64_t)a.rows * heads >= kManyHeads) go(lanes, std::integral_constant<int, 4>{}, std::integral_constant<int, 64>{});
    else go(lanes, std::integral_constant<int, 1>{}, std::integral_constant<int, 8>{});
  };
  const int need = a.cache.d / 16;
  if (need <= 1) by_rows(std::integral_constant<int, 1>{});
  else if (need <= 2) by_rows(std::integral_constant<int, 2>{});
  else if (need <= 4) by_rows(std::integral_constant<int, 4>{});
  else if (need <= 8) by_rows(std::integral_constant<int, 8>{});
  else by_rows(std::integral_constant<int, 16>{});
}

}  // namespace

}  // namespace qtts

int qtts_launch_qkv_to_cache(const qtts::QkvCacheArgs& a, int dtype, hipStream_t st) {
  if (dtype == QTTS_BF16) qtts::launch_qkv<qtts::bf16_t>(a, st);
  else qtts::launch_qkv<qtts::f16_t>(a, st);
  return qtts_check_launch("qkv_to_cache");
}
