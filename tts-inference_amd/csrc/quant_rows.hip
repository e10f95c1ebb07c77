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
#include <algorithm>
#include <type_traits>

#include "common.h"
#include "quant_rows_rule.h"

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

// Codes of four values times c, low first.  int8: one fma onto 1.5 * 2^23, whose low byte is then the
// nearest integer (|v c| <= 127 but for the last bit of c); e4m3: v_cvt_pk_fp8_f32.
template <bool FP8> __device__ __forceinline__ uint32_t codes4(const float* v, float c, bool fin) {
  if constexpr (FP8) {
    int w = __builtin_amdgcn_cvt_pk_fp8_f32(v[0] * c, v[1] * c, 0, false);
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(v[2] * c, v[3] * c, w, true);
  } else {
    uint32_t t[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) t[i] = __float_as_uint(__builtin_fmaf(v[i], c, 12582912.0f));
    const uint32_t lo = __builtin_amdgcn_perm(t[1], t[0], 0x0c0c0400u), hi = __builtin_amdgcn_perm(t[3], t[2], 0x0c0c0400u);
    return fin ? lo | (hi << 16) : 0u;
  }
}

// rms_norm_quant's codes without v's roundings: v / scale = (h w) L / max|h w| where the floor does not hold the scale, so a code
// is the nearest to that quotient, ties (common: h w and max|h w| have few bits) to even.  c = L / max|h w| rounded once breaks every
// tie of a row its own way; with the remainder of that division beside it, h w (hi + lo) is the quotient to 2^-47, rounded once:
// on its tie where it is one, and on the right side of every tie for bf16 rows (no other quotient of theirs is within 2^-24 of one).
// Through inv, the scale and its reciprocal, each rounded, 8 in 10^5 e4m3 codes of bf16 rows were not the nearest; none are.  The
// second product costs 0.04 us a row and nothing where memory binds.
struct NormQuotient {
  float hi, lo;
  bool fin;  // whether the row has a finite scale

  // Of a row with the largest |h w| `top`, code range `limit`.
  __device__ __forceinline__ NormQuotient(float top, float inv, float limit) {
    const float amax = top * inv;
    fin = mag(amax) < 0x7f800000u;
    const bool direct = fin && amax >= kScaleFloor;  // else from inv and the floor (or the NaN or infinity), no tie worth its bits
    hi = (direct ? limit : inv * limit) / (direct ? top : amax < kScaleFloor ? kScaleFloor : amax);
    lo = direct ? __builtin_fmaf(-hi, top, limit) * __builtin_amdgcn_rcpf(top) : 0.0f;
  }

  __device__ __forceinline__ float operator()(float hw) const { return __builtin_fmaf(hw, hi, hw * lo); }
};

// silu(g) = g / (1 + 2^(-g log2 e)), the exponential and the reciprocal by the hardware's (an ulp each; the
// exponent's own rounding makes it |g| ulps where the result is e^-|g| small).  The quotient is taken of g / 16 and 1 / 16 of the
// rest: the reciprocal gives zero for what is under fp32's smallest normal, which 1 / (1 + e^-g) is from g = -87.4 on, silu(g) not.
__device__ __forceinline__ float silu_f32(float g) {
  return g * 0.0625f * __builtin_amdgcn_rcpf(__builtin_fmaf(__builtin_amdgcn_exp2f(-1.44269504f * g), 0.0625f, 0.0625f));
}

// ---- eight elements of a row --------------------------------------------------------------
// VEC: eight neighbours (16-byte aligned, K % 8 == 0), loaded and stored as vectors.  Otherwise element
// i of vector j is column (8 j + i) T + tid: neighbouring lanes on neighbouring elements, one at a time,
// for rows that start anywhere; columns past K read the last one and count as zero.

struct Eight { float f[8]; };

template <typename XT, bool VEC, int T> struct RowAccess {
  int k, tid;

  __device__ __forceinline__ bool live(int j, int i) const {
    return VEC ? 8 * (tid + T * j) < k : (8 * j + i) * T + tid < k;
  }

  __device__ __forceinline__ Eight load(const XT* row, int j) const {
    Eight e;
    if constexpr (VEC && sizeof(XT) == 2) {
      const i32x4_t v = *(const i32x4_t*)(row + min(8 * (tid + T * j), k - 8));  // clamped: in the row
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        e.f[2 * i] = to_f32(XT{(uint16_t)v[i]});
        e.f[2 * i + 1] = to_f32(XT{(uint16_t)((uint32_t)v[i] >> 16)});
      }
    } else if constexpr (VEC) {
      const f32x4_t* v = (const f32x4_t*)(row + min(8 * (tid + T * j), k - 8));
      const f32x4_t lo = v[0], hi = v[1];
#pragma unroll
      for (int i = 0; i < 4; ++i) e.f[i] = lo[i], e.f[4 + i] = hi[i];
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) e.f[i] = to_f32(row[min((8 * j + i) * T + tid, k - 1)]);
    }
    return e;
  }

  __device__ __forceinline__ void store(XT* row, int j, const Eight& e) const {
    if constexpr (VEC) {
      if (!live(j, 0)) return;
      XT* to = row + 8 * (tid + T * j);
      if constexpr (sizeof(XT) == 2) {
        i32x4_t v;
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = (int)pack2_f32<XT>(e.f[2 * i], e.f[2 * i + 1]);
        *(i32x4_t*)to = v;
      } else {
        ((f32x4_t*)to)[0] = f32x4_t{e.f[0], e.f[1], e.f[2], e.f[3]};
        ((f32x4_t*)to)[1] = f32x4_t{e.f[4], e.f[5], e.f[6], e.f[7]};
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (live(j, i)) row[(8 * j + i) * T + tid] = from_f32<XT>(e.f[i]);
    }
  }

  // The codes of e * c; zeros for a row that is not `live` (int8).
  template <bool FP8> __device__ __forceinline__ void store_codes(uint8_t* row, int j, const Eight& e, float c, bool fin) const {
    uint32_t w[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) w[h] = codes4<FP8>(&e.f[4 * h], c, fin);
    if constexpr (VEC) {
      if (live(j, 0)) *(uint2*)(row + 8 * (tid + T * j)) = make_uint2(w[0], w[1]);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (live(j, i)) row[(8 * j + i) * T + tid] = (uint8_t)(w[i >> 2] >> (8 * (i & 3)));
    }
  }
};

// Sum and largest magnitude over a workgroup of T threads, in every thread.  One LDS exchange for both.
template <int T> __device__ __forceinline__ void meet(float& ss, uint32_t& mx, float* sum, uint32_t* top) {
  ss = wave_sum_rows(ss);
  mx = wave_umax(mx);
  if constexpr (T > 64) {
    const int tid = threadIdx.x;
    if ((tid & 63) == 0) sum[tid >> 6] = ss, top[tid >> 6] = mx;
    __syncthreads();
    ss = sum[0], mx = top[0];
#pragma unroll
    for (int i = 1; i < T / 64; ++i) ss += sum[i], mx = umax(mx, top[i]);
  }
}

// The row in registers (K <= 8 T V): one memory round trip and one exchange a row.  max |h w| is taken in the
// same pass as the sum of squares, since inv scales every value alike: max |v| = max |h w| inv, and the codes
// need h w alone (NormQuotient).  A product of two 16-bit values is exact in fp32.
// Bound by memory where rows are many: 8192 x 4096 bf16 with residual and hidden, 7 bytes an element, in 37.6 us (6.3 TB/s; a
// copy of 4 GiB 5.1; 8192 x 4095, element by element, 50.6); 1003 x 2048 fp16 without either in 4.7 (3.9 with the same rows in every
// call, which the Infinity Cache then holds); one row in 2.5 (2.3), its latency.
template <typename XT, bool FP8, bool VEC, int T, int V>
__global__ __launch_bounds__(T) void rms_norm_quant_kernel(
    const XT* x, int64_t ldx, const XT* res, int64_t ldr, const XT* __restrict__ w, int k, float eps,
    uint8_t* __restrict__ q, float* __restrict__ sx, XT* hidden, int64_t ldh, XT* __restrict__ normed, int64_t ldn) {
  __shared__ float sum[T / 64];
  __shared__ uint32_t top[T / 64];
  const int64_t row = blockIdx.x;
  const RowAccess<XT, VEC, T> at{k, (int)threadIdx.x};
  Eight p[V], wt[V];
#pragma unroll
  for (int j = 0; j < V; ++j) p[j] = at.load(x + row * ldx, j);
#pragma unroll
  for (int j = 0; j < V; ++j) wt[j] = at.load(w, j);
  if (res) {
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const Eight r = at.load(res + row * ldr, j);
#pragma unroll
      for (int i = 0; i < 8; ++i) p[j].f[i] = round_through<XT>(p[j].f[i] + r.f[i]);
    }
  }
  if (hidden) {  // each element is read and written by one thread: hidden may be x or the residual
#pragma unroll
    for (int j = 0; j < V; ++j) at.store(hidden + row * ldh, j, p[j]);
  }
  float ss = 0.0f;
  uint32_t mx = 0;
#pragma unroll
  for (int j = 0; j < V; ++j)
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float h = at.live(j, i) ? p[j].f[i] : 0.0f;  // a clamped column may hold its hidden already
      ss = __builtin_fmaf(h, h, ss);
      p[j].f[i] = h * wt[j].f[i];
      mx = umax(mx, mag(p[j].f[i]));
    }
  meet<T>(ss, mx, sum, top);
  const float inv = 1.0f / __builtin_sqrtf(ss / (float)k + eps);
  const float s = row_scale<FP8>(__uint_as_float(mx) * inv);
  const NormQuotient quotient(__uint_as_float(mx), inv, code_limit<FP8>());
#pragma unroll
  for (int j = 0; j < V; ++j) {
    Eight e;
#pragma unroll
    for (int i = 0; i < 8; ++i) e.f[i] = quotient(p[j].f[i]);
    at.template store_codes<FP8>(q + row * k, j, e, 1.0f, quotient.fin);
  }
  if (normed) {
#pragma unroll
    for (int j = 0; j < V; ++j) {
#pragma unroll
      for (int i = 0; i < 8; ++i) p[j].f[i] *= inv;
      at.store(normed + row * ldn, j, p[j]);
    }
  }
  if (threadIdx.x == 0) sx[row] = s;
}

// As above, without the sum: the gate and up values of a row meet in registers.  4096 x 6144 fp16 with act, 7 bytes an element, in
// 28.8 us (6.1 TB/s); 1501 bf16 rows without it, 5 bytes, in 10.7 (4.3; 1501 x 6143, element by element, 12.1); 5 rows in 3.2.
template <typename XT, bool FP8, bool VEC, int T, int V>
__global__ __launch_bounds__(T) void silu_mul_quant_kernel(const XT* __restrict__ gu, int64_t ld, int k,
                                                           uint8_t* __restrict__ q, float* __restrict__ sx,
                                                           XT* __restrict__ act, int64_t lda) {
  __shared__ float sum[T / 64];
  __shared__ uint32_t top[T / 64];
  const int64_t row = blockIdx.x;
  const RowAccess<XT, VEC, T> at{k, (int)threadIdx.x};
  const XT* g = gu + row * ld;
  Eight v[V], u[V];
#pragma unroll
  for (int j = 0; j < V; ++j) v[j] = at.load(g, j);
#pragma unroll
  for (int j = 0; j < V; ++j) u[j] = at.load(g + k, j);
  float none = 0.0f;
  uint32_t mx = 0;
#pragma unroll
  for (int j = 0; j < V; ++j)
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      v[j].f[i] = silu_f32(v[j].f[i]) * u[j].f[i];
      mx = umax(mx, mag(v[j].f[i]));
    }
  meet<T>(none, mx, sum, top);
  const float s = row_scale<FP8>(__uint_as_float(mx)), rs = 1.0f / s;
  const bool fin = mag(s) < 0x7f800000u;
#pragma unroll
  for (int j = 0; j < V; ++j) at.template store_codes<FP8>(q + row * k, j, v[j], rs, fin);
  if (act) {
#pragma unroll
    for (int j = 0; j < V; ++j) at.store(act + row * lda, j, v[j]);
  }
  if (threadIdx.x == 0) sx[row] = s;
}

// Longer rows, and more rows than a grid has workgroups: element by element, the row read twice (the second time from cache).
template <typename XT, bool FP8>
__global__ __launch_bounds__(kRowThreads) void rms_norm_quant_long_kernel(
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
    const float s = row_scale<FP8>(__uint_as_float(mx) * inv);
    const NormQuotient quotient(__uint_as_float(mx), inv, code_limit<FP8>());
    for (int64_t c = tid; c < k; c += kRowThreads) {
      const float h = value(c);  // before hidden, which may be x or the residual, is written
      const float hw = h * to_f32(w[c]);
      if (hidden) hidden[row * ldh + c] = from_f32<XT>(h);
      if (normed) normed[row * ldn + c] = from_f32<XT>(hw * inv);
      q[row * k + c] = code_of<FP8>(quotient(hw), quotient.fin);
    }
    if (tid == 0) sx[row] = s;
  }
}

template <typename XT, bool FP8>
__global__ __launch_bounds__(kRowThreads) void silu_mul_quant_long_kernel(const XT* __restrict__ gu, int64_t ld, int64_t k,
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

constexpr int64_t kMaxRowGrid = 1 << 20;  // workgroups of the long kernels; each takes every gridDim-th row

bool aligned(const void* p, int64_t ld, int64_t esz) { return !p || ((uintptr_t)p % 16 == 0 && ld * esz % 16 == 0); }

// f(vec, T, V) with the row kernel's shape as compile-time constants; false where the long kernel takes the call.
template <typename F> bool by_form(bool vec, const RowForm& form, F&& f) {
  auto shape = [&](auto v) {
    using std::integral_constant;
    switch (form.threads * 16 + form.vectors) {
      case 64 * 16 + 1: f(v, integral_constant<int, 64>{}, integral_constant<int, 1>{}); return true;
      case 128 * 16 + 1: f(v, integral_constant<int, 128>{}, integral_constant<int, 1>{}); return true;
      case 256 * 16 + 1: f(v, integral_constant<int, 256>{}, integral_constant<int, 1>{}); return true;
      case 256 * 16 + 2: f(v, integral_constant<int, 256>{}, integral_constant<int, 2>{}); return true;
      case 256 * 16 + 3: f(v, integral_constant<int, 256>{}, integral_constant<int, 3>{}); return true;
      case 256 * 16 + 4: f(v, integral_constant<int, 256>{}, integral_constant<int, 4>{}); return true;
      case 512 * 16 + 3: f(v, integral_constant<int, 512>{}, integral_constant<int, 3>{}); return true;
      case 512 * 16 + 4: f(v, integral_constant<int, 512>{}, integral_constant<int, 4>{}); return true;
      default: return false;
    }
  };
  return vec ? shape(std::true_type{}) : shape(std::false_type{});
}

template <typename XT, bool FP8>
void launch_norm(const void* x, int64_t ldx, const void* res, int64_t ldr, const void* w, int64_t k, float eps, void* q,
                 float* sx, void* hidden, int64_t ldh, void* normed, int64_t ldn, int64_t m, hipStream_t st) {
  constexpr int64_t e = sizeof(XT);
  const bool vec = k % 8 == 0 && aligned(x, ldx, e) && aligned(res, ldr, e) && aligned(w, 8, e) && aligned(hidden, ldh, e) &&
                   aligned(normed, ldn, e) && (uintptr_t)q % 8 == 0;
  const bool done = by_form(vec, row_form(m, k), [&](auto v, auto t, auto n) {
    qtts::launch(&rms_norm_quant_kernel<XT, FP8, v.value, t.value, n.value>, dim3((unsigned)m), dim3(t.value), 0, st,
                 (const XT*)x, ldx, (const XT*)res, ldr, (const XT*)w, k, eps, (uint8_t*)q, sx, (XT*)hidden, ldh,
                 (XT*)normed, ldn);
  });
  if (!done)
    qtts::launch(&rms_norm_quant_long_kernel<XT, FP8>, dim3((unsigned)std::min(m, kMaxRowGrid)), dim3(kRowThreads), 0, st,
                 (const XT*)x, ldx, (const XT*)res, ldr, (const XT*)w, k, eps, (uint8_t*)q, sx, (XT*)hidden, ldh,
                 (XT*)normed, ldn, m);
}

template <typename XT, bool FP8>
void launch_silu(const void* gu, int64_t ld, int64_t k, void* q, float* sx, void* act, int64_t lda, int64_t m,
                 hipStream_t st) {
  constexpr int64_t e = sizeof(XT);
  const bool vec = k % 8 == 0 && aligned(gu, ld, e) && aligned(act, lda, e) && (uintptr_t)q % 8 == 0;
  const bool done = by_form(vec, row_form(m, k), [&](auto v, auto t, auto n) {
    qtts::launch(&silu_mul_quant_kernel<XT, FP8, v.value, t.value, n.value>, dim3((unsigned)m), dim3(t.value), 0, st,
                 (const XT*)gu, ld, k, (uint8_t*)q, sx, (XT*)act, lda);
  });
  if (!done)
    qtts::launch(&silu_mul_quant_long_kernel<XT, FP8>, dim3((unsigned)std::min(m, kMaxRowGrid)), dim3(kRowThreads), 0, st,
                 (const XT*)gu, ld, k, (uint8_t*)q, sx, (XT*)act, lda, m);
}

// f with the element type and the code kind as types.
template <typename F> void by_types(int x_dtype, int codes, F&& f) {
  auto kind = [&](auto xt) {
    if (codes == QTTS_CODE_E4M3) f(xt, std::true_type{});
    else f(xt, std::false_type{});
  };
  if (x_dtype == QTTS_BF16) kind(bf16_t{});
  else if (x_dtype == QTTS_F16) kind(f16_t{});
  else kind(float{});
}

}  // namespace

int qtts_launch_rms_norm_quant(const void* x, int x_dtype, int64_t m, int64_t k, int64_t ldx, const void* res, int64_t ldr,
                               const void* w, float eps, int codes, void* q, float* sx, void* hidden, int64_t ldh,
                               void* normed, int64_t ldn, hipStream_t st) {
  by_types(x_dtype, codes, [&](auto xt, auto fp8) {
    launch_norm<decltype(xt), fp8.value>(x, ldx, res, ldr, w, k, eps, q, sx, hidden, ldh, normed, ldn, m, st);
  });
  return qtts_check_launch("rms_norm_quant");
}

int qtts_launch_silu_mul_quant(const void* gu, int x_dtype, int64_t m, int64_t k, int64_t ld, int codes, void* q, float* sx,
                               void* act, int64_t lda, hipStream_t st) {
  by_types(x_dtype, codes, [&](auto xt, auto fp8) {
    launch_silu<decltype(xt), fp8.value>(gu, ld, k, q, sx, act, lda, m, st);
  });
  return qtts_check_launch("silu_mul_quant");
}
