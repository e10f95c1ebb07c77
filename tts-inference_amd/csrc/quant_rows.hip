// The producers of a W8A8 linear's input, straight to its per-token codes:
//
//  * rms_norm_quant: h = T(x + residual) (T the activations' type; h = x without a residual),
//    inv = 1 / sqrt(sum h^2 / K + eps), v = (h w) inv;
//  * silu_mul_quant: v = silu(g) u of GatedMLP's fused gate_up output, silu(g) = g / (1 + exp(-g));
//
// then scale = max(max_c |v|, 1e-6) / L (L = 448 for e4m3, 127 for int8) and code = round(v / scale),
// to the nearest code, ties to even.  v stays in fp32 from the 16-bit inputs to the code: the separate
// kernels (rms_norm or silu_mul, then the activation quantizer) round it to 16 bits in between.  A NaN
// among a row's v makes its scale NaN, as torch's amax does; e4m3 codes of such a row are NaN, int8
// codes (which have none) zero.
#include "common.h"

using namespace qtts;

namespace qtts {

constexpr int kRowThreads = 256;
constexpr float kScaleFloor = 1e-6f;

template <bool FP8> constexpr float code_limit() { return FP8 ? 448.0f : 127.0f; }

// The larger magnitude as fp32 bits: NaN above infinity above every number, so that a NaN is kept.
__device__ __forceinline__ uint32_t umax(uint32_t a, uint32_t b) { return a > b ? a : b; }
__device__ __forceinline__ uint32_t mag(float v) { return __float_as_uint(v) & 0x7fffffffu; }

__device__ __forceinline__ uint32_t wave_umax(uint32_t v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v = umax(v, (uint32_t)__shfl_xor((int)v, o, 64));
  return v;
}

// The row's scale from its largest |v|; a NaN stays one.
template <bool FP8> __device__ __forceinline__ float row_scale(float amax) {
  return (amax < kScaleFloor ? kScaleFloor : amax) / code_limit<FP8>();
}

// Code of a quotient; `live` is false in a row without a finite scale.
template <bool FP8> __device__ __forceinline__ uint8_t code_of(float v, bool live) {
  if constexpr (FP8) return (uint8_t)e4m3_encode(v);
  else return live ? (uint8_t)(int8_t)int8_code_of(v) : 0;
}

__device__ __forceinline__ float silu_f32(float g) { return g / (1.0f + expf(-g)); }

// One row a workgroup at a time, element by element, the row read twice.
template <typename XT, bool FP8>
__global__ __launch_bounds__(kRowThreads) void rms_norm_quant_kernel(
    const XT* x, int64_t ldx, const XT* res, int64_t ldr, const XT* __restrict__ w, int64_t k, float eps,
    uint8_t* __restrict__ q, float* __restrict__ sx, XT* hidden, int64_t ldh, XT* __restrict__ normed, int64_t ldn,
    int64_t m) {
  __shared__ float sum[kRowThreads / 64];
  __shared__ uint32_t top[kRowThreads / 64];
  const int tid = threadIdx.x;
  for (int64_t row = blockIdx.x; row < m; row += gridDim.x) {
    auto value = [&](int64_t c) {
      const float a = to_f32(x[row * ldx + c]);
      return res ? round_through<XT>(a + to_f32(res[row * ldr + c])) : a;
    };
    float ss = 0.0f;
    uint32_t mx = 0;
    for (int64_t c = tid; c < k; c += kRowThreads) {
      const float h = value(c);
      ss = __builtin_fmaf(h, h, ss);
      mx = umax(mx, mag(h * to_f32(w[c])));
    }
    ss = wave_sum(ss);
    mx = wave_umax(mx);
    __syncthreads();  // the previous row's readers are done
    if ((tid & 63) == 0) sum[tid >> 6] = ss, top[tid >> 6] = mx;
    __syncthreads();
    ss = (sum[0] + sum[1]) + (sum[2] + sum[3]);
    mx = umax(umax(top[0], top[1]), umax(top[2], top[3]));
    const float inv = 1.0f / __builtin_sqrtf(ss / (float)(k ? k : 1) + eps);
    const float s = row_scale<FP8>(__uint_as_float(mx) * inv), rs = 1.0f / s;
    const bool live = mag(s) < 0x7f800000u;
    for (int64_t c = tid; c < k; c += kRowThreads) {
      const float h = value(c);  // before hidden, which may be x or the residual, is written
      const float v = (h * to_f32(w[c])) * inv;
      if (hidden) hidden[row * ldh + c] = from_f32<XT>(h);
      if (normed) normed[row * ldn + c] = from_f32<XT>(v);
      q[row * k + c] = code_of<FP8>(v * rs, live);
    }
    if (tid == 0) sx[row] = s;
  }
}

template <typename XT, bool FP8>
__global__ __launch_bounds__(kRowThreads) void silu_mul_quant_kernel(const XT* __restrict__ gu, int64_t ld, int64_t k,
                                                                     uint8_t* __restrict__ q, float* __restrict__ sx,
                                                                     XT* __restrict__ act, int64_t lda, int64_t m) {
  __shared__ uint32_t top[kRowThreads / 64];
  const int tid = threadIdx.x;
  for (int64_t row = blockIdx.x; row < m; row += gridDim.x) {
    const XT* g = gu + row * ld;
    uint32_t mx = 0;
    for (int64_t c = tid; c < k; c += kRowThreads) mx = umax(mx, mag(silu_f32(to_f32(g[c])) * to_f32(g[k + c])));
    mx = wave_umax(mx);
    __syncthreads();  // the previous row's readers are done
    if ((tid & 63) == 0) top[tid >> 6] = mx;
    __syncthreads();
    mx = umax(umax(top[0], top[1]), umax(top[2], top[3]));
    const float s = row_scale<FP8>(__uint_as_float(mx)), rs = 1.0f / s;
    const bool live = mag(s) < 0x7f800000u;
    for (int64_t c = tid; c < k; c += kRowThreads) {
      const float v = silu_f32(to_f32(g[c])) * to_f32(g[k + c]);
      if (act) act[row * lda + c] = from_f32<XT>(v);
      q[row * k + c] = code_of<FP8>(v * rs, live);
    }
    if (tid == 0) sx[row] = s;
  }
}

}  // namespace qtts

namespace {

constexpr int64_t kMaxRowGrid = 1 << 20;  // workgroups; each takes every gridDim-th row

template <typename XT>
void norm_by_type(bool fp8, const void* x, int64_t ldx, const void* res, int64_t ldr, const void* w, int64_t k, float eps,
                  void* q, float* sx, void* hidden, int64_t ldh, void* normed, int64_t ldn, int64_t m, hipStream_t st) {
  const dim3 grid((unsigned)(m < kMaxRowGrid ? m : kMaxRowGrid)), block(kRowThreads);
  auto go = [&](auto kernel) {
    qtts::launch(kernel, grid, block, 0, st, (const XT*)x, ldx, (const XT*)res, ldr, (const XT*)w, k, eps, (uint8_t*)q, sx,
                 (XT*)hidden, ldh, (XT*)normed, ldn, m);
  };
  if (fp8) go(&rms_norm_quant_kernel<XT, true>);
  else go(&rms_norm_quant_kernel<XT, false>);
}

template <typename XT>
void silu_by_type(bool fp8, const void* gu, int64_t ld, int64_t k, void* q, float* sx, void* act, int64_t lda, int64_t m,
                  hipStream_t st) {
  const dim3 grid((unsigned)(m < kMaxRowGrid ? m : kMaxRowGrid)), block(kRowThreads);
  auto go = [&](auto kernel) {
    qtts::launch(kernel, grid, block, 0, st, (const XT*)gu, ld, k, (uint8_t*)q, sx, (XT*)act, lda, m);
  };
  if (fp8) go(&silu_mul_quant_kernel<XT, true>);
  else go(&silu_mul_quant_kernel<XT, false>);
}

}  // namespace

int qtts_launch_rms_norm_quant(const void* x, int x_dtype, int64_t m, int64_t k, int64_t ldx, const void* res, int64_t ldr,
                               const void* w, float eps, int codes, void* q, float* sx, void* hidden, int64_t ldh,
                               void* normed, int64_t ldn, hipStream_t st) {
  const bool fp8 = codes == QTTS_CODE_E4M3;
  if (x_dtype == QTTS_BF16) norm_by_type<bf16_t>(fp8, x, ldx, res, ldr, w, k, eps, q, sx, hidden, ldh, normed, ldn, m, st);
  else if (x_dtype == QTTS_F16) norm_by_type<f16_t>(fp8, x, ldx, res, ldr, w, k, eps, q, sx, hidden, ldh, normed, ldn, m, st);
  else norm_by_type<float>(fp8, x, ldx, res, ldr, w, k, eps, q, sx, hidden, ldh, normed, ldn, m, st);
  return qtts_check_launch("rms_norm_quant");
}

int qtts_launch_silu_mul_quant(const void* gu, int x_dtype, int64_t m, int64_t k, int64_t ld, int codes, void* q, float* sx,
                               void* act, int64_t lda, hipStream_t st) {
  const bool fp8 = codes == QTTS_CODE_E4M3;
  if (x_dtype == QTTS_BF16) silu_by_type<bf16_t>(fp8, gu, ld, k, q, sx, act, lda, m, st);
  else if (x_dtype == QTTS_F16) silu_by_type<f16_t>(fp8, gu, ld, k, q, sx, act, lda, m, st);
  else silu_by_type<float>(fp8, gu, ld, k, q, sx, act, lda, m, st);
  return qtts_check_launch("silu_mul_quant");
}
