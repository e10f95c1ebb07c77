// C ABI entry points (include/qtts_amd.h): argument checks, device gating, error
// strings and dispatch to the kernel launchers in pack.hip, w8a16.hip, fp8.hip and
// w8a8_int8.hip.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <atomic>
#include <cstdarg>
#include <cstdio>
#include <cstring>
#include <mutex>
#include <vector>

#include "common.h"
#include "layout.h"
#include "lora.h"
#include "paged.h"
#include "qtts_amd.h"

// Launchers implemented next to their kernels.
int qtts_launch_pack_int8(const void* src, int src_dtype, int64_t n, int64_t k, int64_t ld, int8_t* q,
                          void* scale_out, int scale_dtype, float* scale_f32, int div_mode, hipStream_t st);
int qtts_launch_pack_fp8(const void* src, int src_dtype, int64_t n, int64_t k, int64_t ld, uint8_t* q, float* scale,
                         int div_mode, hipStream_t st);
int qtts_launch_quant_act_fp8(const void* x, int x_dtype, int64_t m, int64_t k, int64_t ld, uint8_t* qx, float* sx,
                              int div_mode, hipStream_t st);
int qtts_launch_w8a16(const void* x, int x_dtype, int64_t m, int64_t k, int64_t ldx, const int8_t* q, int64_t n,
                      int64_t ldq, int layout, const void* scale, int scale_dtype, const void* bias, void* y,
                      int64_t ldy, int algo, void* ws, int64_t ws_bytes, hipStream_t st);
int64_t qtts_w8a16_ws_bytes(int64_t m, int64_t n, int64_t k, int algo);
int qtts_launch_fp8_gemm(const uint8_t* qx, const float* sx, int64_t m, int64_t k, int64_t ldqx, const uint8_t* qw,
                         int64_t n, int64_t ldqw, int layout, const float* sw, const void* bias, void* y,
                         int out_dtype, int64_t ldy, int algo, void* ws, int64_t ws_bytes, hipStream_t st);
int qtts_launch_to_strips(const void* src, int64_t n, int64_t k, int64_t ld, void* dst, int kind, hipStream_t st);
int qtts_launch_from_strips(const void* src, int64_t n, int64_t k, void* dst, int64_t ld, int kind, hipStream_t st);
int qtts_launch_dequant_strips(const void* qs, int codes, int64_t n, int64_t k, const void* scale, int sdt, void* w,
                               int w_dtype, int64_t ldw, hipStream_t st);
int64_t qtts_fp8_gemm_ws_bytes(int64_t m, int64_t n, int64_t k, int algo);
int qtts_fp8_fused_ok(int64_t m, int64_t n, int64_t k, int waves);
int qtts_launch_quant_act_int8(const void* x, int x_dtype, int64_t m, int64_t k, int64_t ld, int8_t* qx, float* sx,
                               int div_mode, hipStream_t st);
int qtts_launch_int8_gemm(const int8_t* qx, const float* sx, int64_t m, int64_t k, int64_t ldqx, const int8_t* qw,
                          int64_t n, int64_t ldqw, int layout, const float* sw, const void* bias, void* y,
                          int out_dtype, int64_t ldy, int algo, void* ws, int64_t ws_bytes, hipStream_t st);
int64_t qtts_int8_gemm_ws_bytes(int64_t m, int64_t n, int64_t k, int algo);
int64_t qtts_fp8w_ws_bytes(int64_t m, int64_t n, int64_t k, int algo);
int qtts_launch_fp8w(const void* x, int x_dtype, int64_t m, int64_t k, int64_t ldx, const uint8_t* qs, int64_t n,
                     const float* scale, const void* bias, void* y, int64_t ldy, int algo, void* ws, int64_t ws_bytes,
                     hipStream_t st);
int qtts_launch_silu_mul(const void* gu, int x_dtype, int64_t m, int64_t k, int64_t ld, void* h, int64_t ldh,
                         hipStream_t st);
int64_t qtts_w8a16_silu_ws_bytes(int64_t m, int64_t n, int64_t k, int algo, int x_dtype);
int qtts_launch_w8a16_silu(const void* gu, int x_dtype, int64_t m, int64_t k, int64_t ld, const int8_t* qs, int64_t n,
                           const void* scale, int sdt, const void* bias, void* y, int64_t ldy, int algo, void* ws,
                           int64_t ws_bytes, hipStream_t st);
int qtts_launch_rms_norm(const void* x, int x_dtype, int64_t m, int64_t k, int64_t ldx, const void* w, float eps,
                         void* y, int64_t ldy, hipStream_t st);
int qtts_launch_w8a16_gate_up_silu(const void* x, int x_dtype, int64_t m, int64_t k, int64_t ldx, int pro,
                                   const void* nw, float eps, const int8_t* qs, int64_t n, const void* scale, int sdt,
                                   const void* bias, void* act, int64_t ldact, int algo, void* ws, int64_t ws_bytes,
                                   hipStream_t st);
int64_t qtts_w8a16_fused_ws_bytes(int64_t m, int64_t n, int64_t k, int algo, int x_dtype);
int qtts_launch_w8a16_fused(const void* x, int x_dtype, int64_t m, int64_t k, int64_t ldx, int pro, const void* nw,
                            float eps, const int8_t* qs, int64_t n, const void* scale, int sdt, const void* bias,
                            const void* res, int64_t ldr, void* y, int64_t ldy, int algo, void* ws, int64_t ws_bytes,
                            hipStream_t st);
int qtts_launch_fp8_linear_fused(const void* x, int x_dtype, int64_t m, int64_t k, int64_t ldx, const uint8_t* qws,
                                 int64_t n, const float* sw, const void* bias, void* y, int64_t ldy, int div_mode,
                                 int waves, hipStream_t st);
int qtts_int8_fused_ok(int64_t m, int64_t n, int64_t k, int waves);
int qtts_launch_int8_linear_fused(const void* x, int x_dtype, int64_t m, int64_t k, int64_t ldx, const int8_t* qws,
                                  int64_t n, const float* sw, const void* bias, void* y, int64_t ldy, int div_mode,
                                  int waves, hipStream_t st);
int qtts_launch_rms_norm_quant(const void* x, int x_dtype, int64_t m, int64_t k, int64_t ldx, const void* res, int64_t ldr,
                               const void* w, float eps, int codes, void* q, float* sx, void* hidden, int64_t ldh,
                               void* normed, int64_t ldn, hipStream_t st);
int qtts_launch_silu_mul_quant(const void* gu, int x_dtype, int64_t m, int64_t k, int64_t ld, int codes, void* q, float* sx,
                               void* act, int64_t lda, hipStream_t st);
int64_t qtts_lora_ws_bytes(int64_t m, int64_t parts, int64_t rank);
int qtts_launch_lora_plan(const int32_t* index, int64_t m, int64_t slots, int32_t* plan, hipStream_t st);
int qtts_launch_lora_add(const qtts::LoraArgs& args, int x_dtype, void* ws, hipStream_t st);
int qtts_launch_paged_step(const qtts::PagedStepArgs& args, hipStream_t st);
int qtts_launch_paged_release(const int32_t* which, int32_t* lengths, const int32_t* table, int requests, int cols,
                              int32_t* free_pages, int pages, int32_t* taken, int page_shift, hipStream_t st);
int qtts_launch_qkv_to_cache(const qtts::QkvCacheArgs& args, int dtype, hipStream_t st);
int qtts_launch_paged_attention(const qtts::PagedAttentionArgs& args, int min_new, int dtype, void* ws, hipStream_t st);
int64_t qtts_paged_attention_ws_bytes(int64_t m, int64_t d);

static thread_local char g_last_error[512] = "";

// The weight policy of the entry point running on this thread (common.h: WeightPolicy).
thread_local int qtts::g_weight_policy = 0;

int qtts_set_error(int status, const char* fmt, ...) {
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(g_last_error, sizeof(g_last_error), fmt, ap);
  va_end(ap);
  return status;
}

int qtts_check_launch(const char* what) {
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) return qtts_set_error(QTTS_ERR_HIP, "%s: launch failed: %s", what, hipGetErrorString(e));
  return QTTS_OK;
}

// ---- kernel timer -----------------------------------------------------------------------
// Armed by qtts_kernel_timer_begin with a fixed pool of event pairs; qtts::launch takes
// the next pair for each launch that is not being captured into a graph.

namespace {
std::mutex g_timer_mu;
std::atomic<bool> g_timer_armed{false};
std::vector<hipEvent_t> g_timer_events;  // start0, stop0, start1, stop1, ...
size_t g_timer_used = 0;
int64_t g_timer_untimed = 0;

void timer_release() {
  for (hipEvent_t e : g_timer_events) (void)hipEventDestroy(e);
  g_timer_events.clear();
  g_timer_used = 0;
}
}  // namespace

bool qtts_timer_slot(hipStream_t st, hipEvent_t* start, hipEvent_t* stop) {
  if (!g_timer_armed.load(std::memory_order_acquire)) return false;
  hipStreamCaptureStatus cs = hipStreamCaptureStatusNone;
  if (hipStreamIsCapturing(st, &cs) != hipSuccess) {
    (void)hipGetLastError();
    return false;
  }
  if (cs != hipStreamCaptureStatusNone) return false;
  std::lock_guard<std::mutex> lock(g_timer_mu);
  if (!g_timer_armed.load(std::memory_order_relaxed)) return false;
  if (g_timer_used + 2 > g_timer_events.size()) {
    g_timer_untimed++;
    return false;
  }
  *start = g_timer_events[g_timer_used];
  *stop = g_timer_events[g_timer_used + 1];
  g_timer_used += 2;
  return true;
}

// ---- device gating: gfx950 only ---------------------------------------------------------

namespace {

constexpr int kMaxDevices = 64;
std::atomic<int> g_dev_state[kMaxDevices];  // 0 unknown, 1 supported, 2 unsupported

bool dtype_ok(int d) { return d == QTTS_F32 || d == QTTS_BF16 || d == QTTS_F16; }
int64_t dtype_size(int d) { return d == QTTS_F32 ? 4 : 2; }
bool div_ok(int d) { return d == QTTS_DIV_DEVICE || d == QTTS_DIV_IEEE; }
bool algo_ok(int a) {
  const int f = a & 0xff;
  return f == QTTS_ALGO_AUTO || f == QTTS_ALGO_SKINNY || f == QTTS_ALGO_TILE;
}
// The families of the W8A16 strip GEMM: the others plus the row-split skinny kernels.
bool algo_ok_rows(int a) {
  const int f = a & 0xff;
  return algo_ok(a) || f == QTTS_ALGO_SKINNY_HALF || f == QTTS_ALGO_SKINNY_QUARTER;
}
int64_t al256(int64_t v) { return (v + 255) & ~(int64_t)255; }

// Whether the byte spans of two [rows, cols] matrices (row strides lda, ldb, elements
// of esz bytes) intersect.
bool ranges_overlap(const void* a, int64_t rows_a, int64_t lda, const void* b, int64_t rows_b, int64_t ldb,
                    int64_t cols, int64_t esz) {
  const uintptr_t a0 = (uintptr_t)a, a1 = a0 + (uintptr_t)(((rows_a - 1) * lda + cols) * esz);
  const uintptr_t b0 = (uintptr_t)b, b1 = b0 + (uintptr_t)(((rows_b - 1) * ldb + cols) * esz);
  return a0 < b1 && b0 < a1;
}

// Floor division for a positive divisor.
int64_t floor_div(int64_t a, int64_t d) { return a >= 0 ? a / d : -((-a + d - 1) / d); }

// Whether an [rows_a, cols_a] matrix at a (row stride lda, elements of esz_a bytes) and an
// [rows_b, cols_b] matrix at b (row stride ldb, elements of esz_b bytes) share a byte.  Row by
// row: two column blocks of one buffer whose rows interleave (x = buf[:, :k], y = buf[:, k:])
// share none.  Row i of a covers [a + i * La, a + i * La + Ca) (La = lda * esz_a, Ca = cols_a *
// esz_a), likewise for b; for each row i of a, the rows j of b that meet it satisfy
// j * Lb in (a + i * La - b - Cb, a + i * La - b + Ca).  The loop runs over a's rows once the
// whole spans are known to intersect; more than 2^22 rows are taken to overlap.
bool spans_overlap(const void* a, int64_t rows_a, int64_t lda, int64_t cols_a, int64_t esz_a, const void* b,
                   int64_t rows_b, int64_t ldb, int64_t cols_b, int64_t esz_b) {
  if (rows_a <= 0 || cols_a <= 0 || rows_b <= 0 || cols_b <= 0) return false;
  const int64_t La = lda * esz_a, Ca = cols_a * esz_a, Lb = ldb * esz_b, Cb = cols_b * esz_b;
  const uintptr_t a0 = (uintptr_t)a, a1 = a0 + (uintptr_t)((rows_a - 1) * La + Ca);
  const uintptr_t b0 = (uintptr_t)b, b1 = b0 + (uintptr_t)((rows_b - 1) * Lb + Cb);
  if (!(a0 < b1 && b0 < a1)) return false;
  if (rows_a > (1 << 22) || La <= 0 || Lb <= 0) return true;
  const int64_t d = (int64_t)(a0 - b0);  // a - b, bytes (the spans intersect, so this is small)
  for (int64_t i = 0; i < rows_a; ++i) {
    const int64_t lo = d + i * La - Cb, hi = d + i * La + Ca;  // open interval for j * Lb
    const int64_t j0 = std::max<int64_t>(floor_div(lo, Lb) + 1, 0);
    if (j0 < rows_b && j0 * Lb < hi) return true;
  }
  return false;
}

// Workspace of the one-call linears: the GEMM's own part (its split-K counter block
// always reserved, so the quantized activations never land on counters that later
// calls expect at zero), then the activation codes and their scales.
int64_t linear_ws(int64_t gemm_ws, int64_t m, int64_t k) {
  return al256(std::max<int64_t>(gemm_ws, qtts::kCounterBytes)) + al256(m * k) + al256(m * 4);
}

int current_device_check() {
  int dev = -1;
  hipError_t e = hipGetDevice(&dev);
  if (e != hipSuccess) return qtts_set_error(QTTS_ERR_UNSUPPORTED, "no HIP device: %s", hipGetErrorString(e));
  if (qtts_device_supported(dev) != 1)
    return qtts_set_error(QTTS_ERR_UNSUPPORTED, "device %d is not a gfx950 (MI355X-class) GPU", dev);
  return QTTS_OK;
}

#define QTTS_REQUIRE(cond, ...) \
  do {                          \
    if (!(cond)) return qtts_set_error(QTTS_ERR_INVALID_ARGUMENT, __VA_ARGS__); \
  } while (0)

#define QTTS_TRY(expr)               \
  do {                               \
    int _s = (expr);                 \
    if (_s != QTTS_OK) return _s;    \
  } while (0)

}  // namespace

extern "C" {

int qtts_abi_version(void) { return QTTS_ABI_VERSION; }

const char* qtts_last_error(void) { return g_last_error; }

int qtts_device_supported(int device) {
  if (device < 0 || device >= kMaxDevices) return 0;
  int s = g_dev_state[device].load(std::memory_order_acquire);
  if (s == 0) {
    hipDeviceProp_t prop;
    if (hipGetDeviceProperties(&prop, device) != hipSuccess) {
      (void)hipGetLastError();
      return 0;
    }
    s = (std::strncmp(prop.gcnArchName, "gfx950", 6) == 0) ? 1 : 2;
    g_dev_state[device].store(s, std::memory_order_release);
  }
  return s == 1 ? 1 : 0;
}

int64_t qtts_workspace_bytes(int op, int64_t m, int64_t n, int64_t k, int algo) {
  const qtts::WeightPolicy policy(algo);  // takes QTTS_ALGO_STREAM out of algo
  const bool rows_ok = op == QTTS_OP_W8A16 || op == QTTS_OP_W8A16_FUSED || op == QTTS_OP_W8A16_SILU;
  // sizes past 2^31 are rejected as every entry point rejects them (and m * k stays in range)
  if (m < 0 || n < 0 || k < 0 || m >= (1ll << 31) || n >= (1ll << 31) || k >= (1ll << 31) ||
      !(rows_ok ? algo_ok_rows(algo) : algo_ok(algo)))
    return qtts_set_error(QTTS_ERR_INVALID_ARGUMENT, "bad workspace query");
  if (m == 0 || n == 0) return 0;
  switch (op) {
    case QTTS_OP_W8A16: return qtts_w8a16_ws_bytes(m, n, k, algo);
    case QTTS_OP_W8A8_FP8: return qtts_fp8_gemm_ws_bytes(m, n, k, algo);
    case QTTS_OP_FP8_LINEAR: return linear_ws(qtts_fp8_gemm_ws_bytes(m, n, k, algo), m, k);
    case QTTS_OP_W8A8_INT8: return qtts_int8_gemm_ws_bytes(m, n, k, algo);
    case QTTS_OP_INT8_LINEAR: return linear_ws(qtts_int8_gemm_ws_bytes(m, n, k, algo), m, k);
    case QTTS_OP_FP8W: return qtts_fp8w_ws_bytes(m, n, k, algo);
    case QTTS_OP_W8A16_SILU: return qtts_w8a16_silu_ws_bytes(m, n, k, algo, QTTS_BF16);
    case QTTS_OP_W8A16_FUSED: return qtts_w8a16_fused_ws_bytes(m, n, k, algo, QTTS_BF16);
    case QTTS_OP_LORA:  // n partitions of rank k
      if (n > QTTS_LORA_MAX_PARTS || k > QTTS_LORA_MAX_RANK)
        return qtts_set_error(QTTS_ERR_INVALID_ARGUMENT, "bad workspace query");
      return qtts_lora_ws_bytes(m, n, k);
    case QTTS_OP_PAGED_ATTENTION:  // m rows a key-value head of k
      if (k > qtts::kPagedMaxDim) return qtts_set_error(QTTS_ERR_INVALID_ARGUMENT, "bad workspace query");
      return qtts_paged_attention_ws_bytes(m, k);
    default: return qtts_set_error(QTTS_ERR_INVALID_ARGUMENT, "unknown op %d", op);
  }
}

int qtts_pack_int8_rowwise(const void* src, int src_dtype, int64_t n, int64_t k, int64_t ld_src, int8_t* q_out,
                           void* scale_out, int scale_dtype, float* scale_f32_out, int div_mode, void* stream) {
  QTTS_REQUIRE(n >= 0 && k >= 0, "pack_int8_rowwise: negative size (n=%lld, k=%lld)", (long long)n, (long long)k);
  QTTS_REQUIRE(dtype_ok(src_dtype) && dtype_ok(scale_dtype), "pack_int8_rowwise: bad dtype code");
  QTTS_REQUIRE(div_ok(div_mode), "pack_int8_rowwise: bad div_mode %d", div_mode);
  QTTS_REQUIRE(ld_src >= k, "pack_int8_rowwise: ld_src %lld < k %lld", (long long)ld_src, (long long)k);
  QTTS_REQUIRE(n < (1ll << 31), "pack_int8_rowwise: n too large");
  if (n == 0) return QTTS_OK;
  QTTS_REQUIRE(scale_out && (k == 0 || (src && q_out)), "pack_int8_rowwise: null pointer");
  QTTS_TRY(current_device_check());
  return qtts_launch_pack_int8(src, src_dtype, n, k, ld_src, q_out, scale_out, scale_dtype, scale_f32_out, div_mode,
                               (hipStream_t)stream);
}

int qtts_pack_fp8_e4m3_rowwise(const void* src, int src_dtype, int64_t n, int64_t k, int64_t ld_src,
                               uint8_t* q_out, float* scale_out, int div_mode, void* stream) {
  QTTS_REQUIRE(n >= 0 && k >= 0, "pack_fp8_e4m3_rowwise: negative size");
  QTTS_REQUIRE(dtype_ok(src_dtype), "pack_fp8_e4m3_rowwise: bad dtype code");
  QTTS_REQUIRE(div_ok(div_mode), "pack_fp8_e4m3_rowwise: bad div_mode %d", div_mode);
  QTTS_REQUIRE(ld_src >= k, "pack_fp8_e4m3_rowwise: ld_src < k");
  QTTS_REQUIRE(n < (1ll << 31), "pack_fp8_e4m3_rowwise: n too large");
  if (n == 0) return QTTS_OK;
  QTTS_REQUIRE(scale_out && (k == 0 || (src && q_out)), "pack_fp8_e4m3_rowwise: null pointer");
  QTTS_TRY(current_device_check());
  return qtts_launch_pack_fp8(src, src_dtype, n, k, ld_src, q_out, scale_out, div_mode, (hipStream_t)stream);
}

int qtts_w8a16_gemm(const void* x, int x_dtype, int64_t m, int64_t k, int64_t ldx, const int8_t* q, int64_t n,
                    int64_t ldq, const void* scale, int scale_dtype, const void* bias, void* y, int64_t ldy, int algo,
                    void* ws, int64_t ws_bytes, void* stream) {
  const qtts::WeightPolicy policy(algo);  // takes QTTS_ALGO_STREAM out of algo
  QTTS_REQUIRE(m >= 0 && n >= 0 && k >= 0, "w8a16_gemm: negative size (m=%lld, n=%lld, k=%lld)", (long long)m,
               (long long)n, (long long)k);
  QTTS_REQUIRE(m < (1ll << 31) && n < (1ll << 31) && k < (1ll << 31), "w8a16_gemm: size too large");
  QTTS_REQUIRE(dtype_ok(x_dtype) && dtype_ok(scale_dtype), "w8a16_gemm: bad dtype code");
  QTTS_REQUIRE(algo_ok(algo), "w8a16_gemm: bad algo %d", algo);
  QTTS_REQUIRE(ldx >= k && ldq >= k && ldy >= n, "w8a16_gemm: leading dimension smaller than the row");
  QTTS_REQUIRE(ws_bytes >= 0, "w8a16_gemm: negative workspace size");
  if (m == 0 || n == 0) return QTTS_OK;
  QTTS_REQUIRE(scale && y && (k == 0 || (x && q)), "w8a16_gemm: null pointer");
  // Every workgroup reads all x rows of its K range while others write y.
  QTTS_REQUIRE(!spans_overlap(x, m, ldx, k, dtype_size(x_dtype), y, m, ldy, n, dtype_size(x_dtype)),
               "w8a16_gemm: y overlaps x");
  QTTS_TRY(current_device_check());
  return qtts_launch_w8a16(x, x_dtype, m, k, ldx, q, n, ldq, qtts::kLayoutRowMajor, scale, scale_dtype, bias, y, ldy,
                           algo, ws, ws_bytes, (hipStream_t)stream);
}

int qtts_w8a16_gemm_strips(const void* x, int x_dtype, int64_t m, int64_t k, int64_t ldx, const int8_t* qs, int64_t n,
                           const void* scale, int scale_dtype, const void* bias, void* y, int64_t ldy, int algo,
                           void* ws, int64_t ws_bytes, void* stream) {
  const qtts::WeightPolicy policy(algo);  // takes QTTS_ALGO_STREAM out of algo
  QTTS_REQUIRE(m >= 0 && n >= 0 && k >= 0, "w8a16_gemm_strips: negative size (m=%lld, n=%lld, k=%lld)", (long long)m,
               (long long)n, (long long)k);
  QTTS_REQUIRE(m < (1ll << 31) && n < (1ll << 31) && k < (1ll << 31), "w8a16_gemm_strips: size too large");
  QTTS_REQUIRE(dtype_ok(x_dtype) && dtype_ok(scale_dtype), "w8a16_gemm_strips: bad dtype code");
  QTTS_REQUIRE(algo_ok_rows(algo), "w8a16_gemm_strips: bad algo %d", algo);
  QTTS_REQUIRE(ldx >= k && ldy >= n, "w8a16_gemm_strips: leading dimension smaller than the row");
  QTTS_REQUIRE(ws_bytes >= 0, "w8a16_gemm_strips: negative workspace size");
  if (m == 0 || n == 0) return QTTS_OK;
  QTTS_REQUIRE(scale && y && x && qs, "w8a16_gemm_strips: null pointer");
  QTTS_REQUIRE(!spans_overlap(x, m, ldx, k, dtype_size(x_dtype), y, m, ldy, n, dtype_size(x_dtype)),
               "w8a16_gemm_strips: y overlaps x");
  QTTS_TRY(current_device_check());
  return qtts_launch_w8a16(x, x_dtype, m, k, ldx, qs, n, 0, qtts::kLayoutStrips, scale, scale_dtype, bias, y, ldy,
                           algo, ws, ws_bytes, (hipStream_t)stream);
}

int qtts_quant_act_fp8_rows(const void* x, int x_dtype, int64_t m, int64_t k, int64_t ldx, uint8_t* qx, float* sx,
                            int div_mode, void* stream) {
  QTTS_REQUIRE(m >= 0 && k >= 0, "quant_act_fp8_rows: negative size");
  QTTS_REQUIRE(m < (1ll << 31), "quant_act_fp8_rows: m too large");
  QTTS_REQUIRE(dtype_ok(x_dtype), "quant_act_fp8_rows: bad dtype code");
  QTTS_REQUIRE(div_ok(div_mode), "quant_act_fp8_rows: bad div_mode %d", div_mode);
  QTTS_REQUIRE(ldx >= k, "quant_act_fp8_rows: ldx < k");
  if (m == 0) return QTTS_OK;
  QTTS_REQUIRE(sx && (k == 0 || (x && qx)), "quant_act_fp8_rows: null pointer");
  QTTS_TRY(current_device_check());
  return qtts_launch_quant_act_fp8(x, x_dtype, m, k, ldx, qx, sx, div_mode, (hipStream_t)stream);
}

int qtts_w8a8_fp8_gemm(const uint8_t* qx, const float* sx, int64_t m, int64_t k, int64_t ldqx, const uint8_t* qw,
                       int64_t n, int64_t ldqw, const float* sw, const void* bias, void* y, int out_dtype,
                       int64_t ldy, int algo, void* ws, int64_t ws_bytes, void* stream) {
  const qtts::WeightPolicy policy(algo);  // takes QTTS_ALGO_STREAM out of algo
  QTTS_REQUIRE(m >= 0 && n >= 0 && k >= 0, "w8a8_fp8_gemm: negative size");
  QTTS_REQUIRE(m < (1ll << 31) && n < (1ll << 31) && k < (1ll << 31), "w8a8_fp8_gemm: size too large");
  QTTS_REQUIRE(dtype_ok(out_dtype), "w8a8_fp8_gemm: bad dtype code");
  QTTS_REQUIRE(algo_ok(algo), "w8a8_fp8_gemm: bad algo %d", algo);
  QTTS_REQUIRE(ldqx >= k && ldqw >= k && ldy >= n, "w8a8_fp8_gemm: leading dimension smaller than the row");
  QTTS_REQUIRE(ws_bytes >= 0, "w8a8_fp8_gemm: negative workspace size");
  if (m == 0 || n == 0) return QTTS_OK;
  QTTS_REQUIRE(sx && sw && y && (k == 0 || (qx && qw)), "w8a8_fp8_gemm: null pointer");
  QTTS_REQUIRE(!spans_overlap(qx, m, ldqx, k, 1, y, m, ldy, n, dtype_size(out_dtype)), "w8a8_fp8_gemm: y overlaps qx");
  QTTS_TRY(current_device_check());
  return qtts_launch_fp8_gemm(qx, sx, m, k, ldqx, qw, n, ldqw, qtts::kLayoutRowMajor, sw, bias, y, out_dtype, ldy,
                              algo, ws, ws_bytes, (hipStream_t)stream);
}

int qtts_w8a8_fp8_gemm_strips(const uint8_t* qx, const float* sx, int64_t m, int64_t k, int64_t ldqx,
                              const uint8_t* qws, int64_t n, const float* sw, const void* bias, void* y, int out_dtype,
                              int64_t ldy, int algo, void* ws, int64_t ws_bytes, void* stream) {
  const qtts::WeightPolicy policy(algo);  // takes QTTS_ALGO_STREAM out of algo
  QTTS_REQUIRE(m >= 0 && n >= 0 && k >= 0, "w8a8_fp8_gemm_strips: negative size");
  QTTS_REQUIRE(m < (1ll << 31) && n < (1ll << 31) && k < (1ll << 31), "w8a8_fp8_gemm_strips: size too large");
  QTTS_REQUIRE(dtype_ok(out_dtype), "w8a8_fp8_gemm_strips: bad dtype code");
  QTTS_REQUIRE(algo_ok(algo), "w8a8_fp8_gemm_strips: bad algo %d", algo);
  QTTS_REQUIRE(ldqx >= k && ldy >= n, "w8a8_fp8_gemm_strips: leading dimension smaller than the row");
  QTTS_REQUIRE(ws_bytes >= 0, "w8a8_fp8_gemm_strips: negative workspace size");
  if (m == 0 || n == 0) return QTTS_OK;
  QTTS_REQUIRE(qx && sx && qws && sw && y, "w8a8_fp8_gemm_strips: null pointer");
  QTTS_REQUIRE(!spans_overlap(qx, m, ldqx, k, 1, y, m, ldy, n, dtype_size(out_dtype)),
               "w8a8_fp8_gemm_strips: y overlaps qx");
  QTTS_TRY(current_device_check());
  return qtts_launch_fp8_gemm(qx, sx, m, k, ldqx, qws, n, 0, qtts::kLayoutStrips, sw, bias, y, out_dtype, ldy, algo,
                              ws, ws_bytes, (hipStream_t)stream);
}

static int fp8_linear_impl(const void* x, int x_dtype, int64_t m, int64_t k, int64_t ldx, const uint8_t* qw,
                           int64_t n, int64_t ldqw, int layout, const float* sw, const void* bias, void* y,
                           int64_t ldy, int div_mode, int algo, void* ws, int64_t ws_bytes, void* stream) {
  QTTS_REQUIRE(m >= 0 && n >= 0 && k >= 0, "fp8_linear: negative size");
  QTTS_REQUIRE(m < (1ll << 31) && n < (1ll << 31) && k < (1ll << 31), "fp8_linear: size too large");
  QTTS_REQUIRE(dtype_ok(x_dtype), "fp8_linear: bad dtype code");
  QTTS_REQUIRE(div_ok(div_mode), "fp8_linear: bad div_mode %d", div_mode);
  QTTS_REQUIRE(algo_ok(algo), "fp8_linear: bad algo %d", algo);
  QTTS_REQUIRE(ldx >= k && (layout == qtts::kLayoutStrips || ldqw >= k) && ldy >= n,
               "fp8_linear: leading dimension smaller than the row");
  QTTS_REQUIRE(ws_bytes >= 0, "fp8_linear: negative workspace size");
  if (m == 0 || n == 0) return QTTS_OK;
  QTTS_REQUIRE(sw && y && (k == 0 || (x && qw)), "fp8_linear: null pointer");
  // The decode kernel has every workgroup read all of x while others write y.
  QTTS_REQUIRE(!spans_overlap(x, m, ldx, k, dtype_size(x_dtype), y, m, ldy, n, dtype_size(x_dtype)),
               "fp8_linear: y overlaps x");
  // Decode rows on strip weights: quantization fused into the GEMM, one kernel, no
  // workspace.  A wave count alone (family SKINNY or AUTO, no split count or chunk
  // count) sets the fused kernel's waves; an explicit split count keeps the two-kernel path.
  const int fused_waves = (algo >> 16) & 0xff;
  if (layout == qtts::kLayoutStrips && (algo & 0xff) != QTTS_ALGO_TILE && ((algo >> 8) & 0xff) == 0 &&
      (algo >> 24) == 0 && x_dtype != QTTS_F32 && (uintptr_t)x % 16 == 0 && ldx % 8 == 0 &&
      qtts_fp8_fused_ok(m, n, k, fused_waves)) {
    QTTS_TRY(current_device_check());
    return qtts_launch_fp8_linear_fused(x, x_dtype, m, k, ldx, qw, n, sw, bias, y, ldy, div_mode, fused_waves,
                                        (hipStream_t)stream);
  }
  // Layout: the GEMM's own workspace (split-K counters first) from the start, the
  // quantized activations and their scales at the end.
  const int64_t qx_bytes = al256(m * k), sx_bytes = al256(m * 4);
  const int64_t need = linear_ws(qtts_fp8_gemm_ws_bytes(m, n, k, algo), m, k);
  QTTS_REQUIRE(ws != nullptr, "fp8_linear: a workspace of %lld bytes is required", (long long)need);
  if (ws_bytes < qtts::kCounterBytes + qx_bytes + sx_bytes)
    return qtts_set_error(QTTS_ERR_WORKSPACE, "fp8_linear: workspace of %lld bytes < %lld needed", (long long)ws_bytes,
                          (long long)need);
  const int64_t tail = (ws_bytes - qx_bytes - sx_bytes) & ~(int64_t)255;
  QTTS_TRY(current_device_check());
  uint8_t* qx = (uint8_t*)ws + tail;
  float* sx = (float*)((char*)ws + tail + qx_bytes);
  QTTS_TRY(qtts_launch_quant_act_fp8(x, x_dtype, m, k, ldx, qx, sx, div_mode, (hipStream_t)stream));
  return qtts_launch_fp8_gemm(qx, sx, m, k, k, qw, n, ldqw, layout, sw, bias, y, x_dtype, ldy, algo,
                              tail > 0 ? ws : nullptr, tail, (hipStream_t)stream);
}

int qtts_fp8_linear(const void* x, int x_dtype, int64_t m, int64_t k, int64_t ldx, const uint8_t* qw, int64_t n,
                    int64_t ldqw, const float* sw, const void* bias, void* y, int64_t ldy, int div_mode, int algo,
                    void* ws, int64_t ws_bytes, void* stream) {
  const qtts::WeightPolicy policy(algo);  // takes QTTS_ALGO_STREAM out of algo
  return fp8_linear_impl(x, x_dtype, m, k, ldx, qw, n, ldqw, qtts::kLayoutRowMajor, sw, bias, y, ldy, div_mode, algo, ws,
                         ws_bytes, stream);
}

int qtts_fp8_linear_strips(const void* x, int x_dtype, int64_t m, int64_t k, int64_t ldx, const uint8_t* qws,
                           int64_t n, const float* sw, const void* bias, void* y, int64_t ldy, int div_mode, int algo,
                           void* ws, int64_t ws_bytes, void* stream) {
  const qtts::WeightPolicy policy(algo);  // takes QTTS_ALGO_STREAM out of algo
  return fp8_linear_impl(x, x_dtype, m, k, ldx, qws, n, 0, qtts::kLayoutStrips, sw, bias, y, ldy, div_mode, algo, ws,
                         ws_bytes, stream);
}

}  // extern "C"

// ---- the fp8 linear on a library-owned workspace (qtts_fp8_linear_strips_static) ---------
// `scratch` is that workspace: one array per GPU, kept until the process ends.  In host code
// its name is a host-side stand-in, never a device address; the device address of each
// GPU's copy comes from hipGetSymbolAddress, with that GPU current, and only that address
// is handed to kernels.
static __device__ __align__(256) unsigned char scratch[QTTS_STATIC_SCRATCH_BYTES];

namespace {
std::mutex g_scratch_mu;
void* g_scratch_ptr[kMaxDevices] = {};

__global__ void zero_words_kernel(uint32_t* p, int n) {
  const int i = blockIdx.x * blockDim.x + threadIdx.x;
  if (i < n) p[i] = 0u;
}

// The current GPU's scratch address, resolved once per GPU.  On that first call the split-K
// counter block at its start is cleared with a kernel on `st` (the loader zero-fills the
// array too; every later call leaves the counters at zero again).
int scratch_of_current_device(hipStream_t st, void** out) {
  int dev = -1;
  hipError_t e = hipGetDevice(&dev);
  if (e != hipSuccess) return qtts_set_error(QTTS_ERR_UNSUPPORTED, "no HIP device: %s", hipGetErrorString(e));
  if (dev < 0 || dev >= kMaxDevices) return qtts_set_error(QTTS_ERR_UNSUPPORTED, "device %d out of range", dev);
  std::lock_guard<std::mutex> lock(g_scratch_mu);
  if (!g_scratch_ptr[dev]) {
    void* p = nullptr;
    e = hipGetSymbolAddress(&p, HIP_SYMBOL(scratch));
    if (e != hipSuccess || !p)
      return qtts_set_error(QTTS_ERR_HIP, "static scratch: hipGetSymbolAddress failed on device %d: %s", dev,
                            hipGetErrorString(e));
    const int words = (int)(qtts::kCounterBytes / 4);
    qtts::launch(zero_words_kernel, dim3((words + 255) / 256), dim3(256), 0, st, (uint32_t*)p, words);
    QTTS_TRY(qtts_check_launch("static scratch clear"));
    g_scratch_ptr[dev] = p;
  }
  *out = g_scratch_ptr[dev];
  return QTTS_OK;
}
}  // namespace

extern "C" {

int qtts_fp8_linear_strips_static(const void* x, int x_dtype, int64_t m, int64_t k, int64_t ldx, const uint8_t* qws,
                                  int64_t n, const float* sw, const void* bias, void* y, int64_t ldy, int div_mode,
                                  int algo, void* stream) {
  const qtts::WeightPolicy policy(algo);  // takes QTTS_ALGO_STREAM out of algo
  QTTS_REQUIRE(m >= 0 && n >= 0 && k >= 0, "fp8_linear_strips_static: negative size");
  QTTS_REQUIRE(m < (1ll << 31) && k < (1ll << 31), "fp8_linear_strips_static: size too large");
  // The activation codes, their scales and the counter block must fit; a split-K choice that
  // does not fit in what is left runs without the split.
  const int64_t least = qtts::kCounterBytes + al256(m * k) + al256(m * 4);
  if (least > QTTS_STATIC_SCRATCH_BYTES)
    return qtts_set_error(QTTS_ERR_WORKSPACE,
                          "fp8_linear_strips_static: m * k = %lld activation bytes need %lld workspace bytes, "
                          "more than the %lld of the static scratch",
                          (long long)(m * k), (long long)least, (long long)QTTS_STATIC_SCRATCH_BYTES);
  if (m == 0 || n == 0) return fp8_linear_impl(x, x_dtype, m, k, ldx, qws, n, 0, qtts::kLayoutStrips, sw, bias, y,
                                               ldy, div_mode, algo, nullptr, 0, stream);
  QTTS_TRY(current_device_check());
  void* ws = nullptr;
  QTTS_TRY(scratch_of_current_device((hipStream_t)stream, &ws));
  return fp8_linear_impl(x, x_dtype, m, k, ldx, qws, n, 0, qtts::kLayoutStrips, sw, bias, y, ldy, div_mode, algo, ws,
                         QTTS_STATIC_SCRATCH_BYTES, stream);
}

int qtts_quant_act_int8_rows(const void* x, int x_dtype, int64_t m, int64_t k, int64_t ldx, int8_t* qx, float* sx,
                             int div_mode, void* stream) {
  QTTS_REQUIRE(m >= 0 && k >= 0, "quant_act_int8_rows: negative size");
  QTTS_REQUIRE(m < (1ll << 31), "quant_act_int8_rows: m too large");
  QTTS_REQUIRE(dtype_ok(x_dtype), "quant_act_int8_rows: bad dtype code");
  QTTS_REQUIRE(div_ok(div_mode), "quant_act_int8_rows: bad div_mode %d", div_mode);
  QTTS_REQUIRE(ldx >= k, "quant_act_int8_rows: ldx < k");
  if (m == 0) return QTTS_OK;
  QTTS_REQUIRE(sx && (k == 0 || (x && qx)), "quant_act_int8_rows: null pointer");
  QTTS_TRY(current_device_check());
  return qtts_launch_quant_act_int8(x, x_dtype, m, k, ldx, qx, sx, div_mode, (hipStream_t)stream);
}

static int int8_gemm_impl(const char* what, const int8_t* qx, const float* sx, int64_t m, int64_t k, int64_t ldqx,
                          const int8_t* qw, int64_t n, int64_t ldqw, int layout, const float* sw, const void* bias,
                          void* y, int out_dtype, int64_t ldy, int algo, void* ws, int64_t ws_bytes, void* stream) {
  QTTS_REQUIRE(m >= 0 && n >= 0 && k >= 0, "%s: negative size", what);
  QTTS_REQUIRE(m < (1ll << 31) && n < (1ll << 31) && k < (1ll << 31), "%s: size too large", what);
  QTTS_REQUIRE(dtype_ok(out_dtype), "%s: bad dtype code", what);
  QTTS_REQUIRE(algo_ok(algo), "%s: bad algo %d", what, algo);
  QTTS_REQUIRE(ldqx >= k && (layout == qtts::kLayoutStrips || ldqw >= k) && ldy >= n,
               "%s: leading dimension smaller than the row", what);
  QTTS_REQUIRE(ws_bytes >= 0, "%s: negative workspace size", what);
  if (m == 0 || n == 0) return QTTS_OK;
  QTTS_REQUIRE(sx && sw && y && (k == 0 || (qx && qw)), "%s: null pointer", what);
  QTTS_REQUIRE(!spans_overlap(qx, m, ldqx, k, 1, y, m, ldy, n, dtype_size(out_dtype)), "%s: y overlaps qx", what);
  QTTS_TRY(current_device_check());
  return qtts_launch_int8_gemm(qx, sx, m, k, ldqx, qw, n, ldqw, layout, sw, bias, y, out_dtype, ldy, algo, ws, ws_bytes,
                               (hipStream_t)stream);
}

int qtts_w8a8_int8_gemm(const int8_t* qx, const float* sx, int64_t m, int64_t k, int64_t ldqx, const int8_t* qw,
                        int64_t n, int64_t ldqw, const float* sw, const void* bias, void* y, int out_dtype,
                        int64_t ldy, int algo, void* ws, int64_t ws_bytes, void* stream) {
  const qtts::WeightPolicy policy(algo);  // takes QTTS_ALGO_STREAM out of algo
  return int8_gemm_impl("w8a8_int8_gemm", qx, sx, m, k, ldqx, qw, n, ldqw, qtts::kLayoutRowMajor, sw, bias, y,
                        out_dtype, ldy, algo, ws, ws_bytes, stream);
}

int qtts_w8a8_int8_gemm_strips(const int8_t* qx, const float* sx, int64_t m, int64_t k, int64_t ldqx,
                               const int8_t* qws, int64_t n, const float* sw, const void* bias, void* y, int out_dtype,
                               int64_t ldy, int algo, void* ws, int64_t ws_bytes, void* stream) {
  const qtts::WeightPolicy policy(algo);  // takes QTTS_ALGO_STREAM out of algo
  return int8_gemm_impl("w8a8_int8_gemm_strips", qx, sx, m, k, ldqx, qws, n, 0, qtts::kLayoutStrips, sw, bias, y,
                        out_dtype, ldy, algo, ws, ws_bytes, stream);
}

static int int8_linear_impl(const void* x, int x_dtype, int64_t m, int64_t k, int64_t ldx, const int8_t* qw,
                            int64_t n, int64_t ldqw, int layout, const float* sw, const void* bias, void* y,
                            int64_t ldy, int div_mode, int algo, void* ws, int64_t ws_bytes, void* stream) {
  QTTS_REQUIRE(m >= 0 && n >= 0 && k >= 0, "int8_linear: negative size");
  QTTS_REQUIRE(m < (1ll << 31) && n < (1ll << 31) && k < (1ll << 31), "int8_linear: size too large");
  QTTS_REQUIRE(dtype_ok(x_dtype), "int8_linear: bad dtype code");
  QTTS_REQUIRE(div_ok(div_mode), "int8_linear: bad div_mode %d", div_mode);
  QTTS_REQUIRE(algo_ok(algo), "int8_linear: bad algo %d", algo);
  QTTS_REQUIRE(ldx >= k && (layout == qtts::kLayoutStrips || ldqw >= k) && ldy >= n,
               "int8_linear: leading dimension smaller than the row");
  QTTS_REQUIRE(ws_bytes >= 0, "int8_linear: negative workspace size");
  if (m == 0 || n == 0) return QTTS_OK;
  QTTS_REQUIRE(sw && y && (k == 0 || (x && qw)), "int8_linear: null pointer");
  // The decode kernel has every workgroup read all of x while others write y.
  QTTS_REQUIRE(!spans_overlap(x, m, ldx, k, dtype_size(x_dtype), y, m, ldy, n, dtype_size(x_dtype)),
               "int8_linear: y overlaps x");
  // Decode rows on strip weights: quantization fused into the GEMM, one kernel, no
  // workspace.  A wave count alone (family SKINNY or AUTO, no split count or chunk
  // count) sets the fused kernel's waves; an explicit split count keeps the two-kernel path.
  const int fused_waves = (algo >> 16) & 0xff;
  if (layout == qtts::kLayoutStrips && (algo & 0xff) != QTTS_ALGO_TILE && ((algo >> 8) & 0xff) == 0 &&
      (algo >> 24) == 0 && x_dtype != QTTS_F32 && (uintptr_t)x % 16 == 0 && ldx % 8 == 0 &&
      qtts_int8_fused_ok(m, n, k, fused_waves)) {
    QTTS_TRY(current_device_check());
    return qtts_launch_int8_linear_fused(x, x_dtype, m, k, ldx, qw, n, sw, bias, y, ldy, div_mode, fused_waves,
                                         (hipStream_t)stream);
  }
  // Layout: the GEMM's own workspace (split-K counters first) from the start, the
  // quantized activations (rows of k bytes, 16-byte aligned when k % 16 == 0) and
  // their scales at the end.
  const int64_t qx_bytes = al256(m * k), sx_bytes = al256(m * 4);
  const int64_t need = linear_ws(qtts_int8_gemm_ws_bytes(m, n, k, algo), m, k);
  QTTS_REQUIRE(ws != nullptr, "int8_linear: a workspace of %lld bytes is required", (long long)need);
  if (ws_bytes < qtts::kCounterBytes + qx_bytes + sx_bytes)
    return qtts_set_error(QTTS_ERR_WORKSPACE, "int8_linear: workspace of %lld bytes < %lld needed", (long long)ws_bytes,
                          (long long)need);
  const int64_t tail = (ws_bytes - qx_bytes - sx_bytes) & ~(int64_t)255;
  QTTS_TRY(current_device_check());
  int8_t* qx = (int8_t*)ws + tail;
  float* sx = (float*)((char*)ws + tail + qx_bytes);
  QTTS_TRY(qtts_launch_quant_act_int8(x, x_dtype, m, k, ldx, qx, sx, div_mode, (hipStream_t)stream));
  return qtts_launch_int8_gemm(qx, sx, m, k, k, qw, n, ldqw, layout, sw, bias, y, x_dtype, ldy, algo,
                               tail > 0 ? ws : nullptr, tail, (hipStream_t)stream);
}

int qtts_int8_linear(const void* x, int x_dtype, int64_t m, int64_t k, int64_t ldx, const int8_t* qw, int64_t n,
                     int64_t ldqw, const float* sw, const void* bias, void* y, int64_t ldy, int div_mode, int algo,
                     void* ws, int64_t ws_bytes, void* stream) {
  const qtts::WeightPolicy policy(algo);  // takes QTTS_ALGO_STREAM out of algo
  return int8_linear_impl(x, x_dtype, m, k, ldx, qw, n, ldqw, qtts::kLayoutRowMajor, sw, bias, y, ldy, div_mode, algo,
                          ws, ws_bytes, stream);
}

int qtts_int8_linear_strips(const void* x, int x_dtype, int64_t m, int64_t k, int64_t ldx, const int8_t* qws,
                            int64_t n, const float* sw, const void* bias, void* y, int64_t ldy, int div_mode, int algo,
                            void* ws, int64_t ws_bytes, void* stream) {
  const qtts::WeightPolicy policy(algo);  // takes QTTS_ALGO_STREAM out of algo
  return int8_linear_impl(x, x_dtype, m, k, ldx, qws, n, 0, qtts::kLayoutStrips, sw, bias, y, ldy, div_mode, algo, ws,
                          ws_bytes, stream);
}

int qtts_silu_mul(const void* gate_up, int x_dtype, int64_t m, int64_t k, int64_t ld_gate_up, void* h, int64_t ldh,
                  void* stream) {
  QTTS_REQUIRE(m >= 0 && k >= 0, "silu_mul: negative size");
  QTTS_REQUIRE(m < 65536 && k < (1ll << 31), "silu_mul: size too large");
  QTTS_REQUIRE(dtype_ok(x_dtype), "silu_mul: bad dtype code");
  QTTS_REQUIRE(ld_gate_up >= 2 * k && ldh >= k, "silu_mul: leading dimension smaller than the row");
  if (m == 0 || k == 0) return QTTS_OK;
  QTTS_REQUIRE(gate_up && h, "silu_mul: null pointer");
  QTTS_TRY(current_device_check());
  return qtts_launch_silu_mul(gate_up, x_dtype, m, k, ld_gate_up, h, ldh, (hipStream_t)stream);
}

int qtts_w8a16_silu_mul_gemm_strips(const void* gate_up, int x_dtype, int64_t m, int64_t k, int64_t ld_gate_up,
                                    const int8_t* qs, int64_t n, const void* scale, int scale_dtype, const void* bias,
                                    void* y, int64_t ldy, int algo, void* ws, int64_t ws_bytes, void* stream) {
  const qtts::WeightPolicy policy(algo);  // takes QTTS_ALGO_STREAM out of algo
  QTTS_REQUIRE(m >= 0 && n >= 0 && k >= 0, "w8a16_silu_mul_gemm_strips: negative size");
  QTTS_REQUIRE(m < 65536 && n < (1ll << 31) && k < (1ll << 30), "w8a16_silu_mul_gemm_strips: size too large");
  QTTS_REQUIRE(x_dtype == QTTS_BF16 || x_dtype == QTTS_F16, "w8a16_silu_mul_gemm_strips: activations must be bf16 or fp16");
  QTTS_REQUIRE(dtype_ok(scale_dtype), "w8a16_silu_mul_gemm_strips: bad scale dtype code");
  QTTS_REQUIRE(algo_ok_rows(algo), "w8a16_silu_mul_gemm_strips: bad algo %d", algo);
  QTTS_REQUIRE(k % 16 == 0, "w8a16_silu_mul_gemm_strips: K %% 16 != 0 (K=%lld)", (long long)k);
  QTTS_REQUIRE(ld_gate_up >= 2 * k && ldy >= n, "w8a16_silu_mul_gemm_strips: leading dimension smaller than the row");
  QTTS_REQUIRE(ws_bytes >= 0, "w8a16_silu_mul_gemm_strips: negative workspace size");
  if (m == 0 || n == 0) return QTTS_OK;
  QTTS_REQUIRE(gate_up && qs && scale && y, "w8a16_silu_mul_gemm_strips: null pointer");
  QTTS_REQUIRE(!spans_overlap(gate_up, m, ld_gate_up, 2 * k, 2, y, m, ldy, n, 2),
               "w8a16_silu_mul_gemm_strips: y overlaps gate_up");
  QTTS_TRY(current_device_check());
  return qtts_launch_w8a16_silu(gate_up, x_dtype, m, k, ld_gate_up, qs, n, scale, scale_dtype, bias, y, ldy, algo, ws,
                                ws_bytes, (hipStream_t)stream);
}

int qtts_rms_norm(const void* x, int x_dtype, int64_t m, int64_t k, int64_t ldx, const void* weight, float eps, void* y,
                  int64_t ldy, void* stream) {
  QTTS_REQUIRE(m >= 0 && k >= 0, "rms_norm: negative size");
  QTTS_REQUIRE(m < (1ll << 31) && k < (1ll << 31), "rms_norm: size too large");
  QTTS_REQUIRE(dtype_ok(x_dtype), "rms_norm: bad dtype code");
  QTTS_REQUIRE(ldx >= k && ldy >= k, "rms_norm: leading dimension smaller than the row");
  if (m == 0 || k == 0) return QTTS_OK;
  QTTS_REQUIRE(x && weight && y, "rms_norm: null pointer");
  QTTS_TRY(current_device_check());
  return qtts_launch_rms_norm(x, x_dtype, m, k, ldx, weight, eps, y, ldy, (hipStream_t)stream);
}

int qtts_rms_norm_quant(const void* x, int x_dtype, int64_t m, int64_t k, int64_t ldx, const void* residual, int64_t ldr,
                        const void* weight, float eps, int codes, void* qx, float* sx, void* hidden, int64_t ldh,
                        void* normed, int64_t ldn, void* stream) {
  QTTS_REQUIRE(m >= 0 && k >= 0, "rms_norm_quant: negative size");
  QTTS_REQUIRE(m < (1ll << 31) && k < (1ll << 31), "rms_norm_quant: size too large");
  QTTS_REQUIRE(dtype_ok(x_dtype), "rms_norm_quant: bad dtype code");
  QTTS_REQUIRE(codes == QTTS_CODE_INT8 || codes == QTTS_CODE_E4M3, "rms_norm_quant: bad code kind %d", codes);
  QTTS_REQUIRE(ldx >= k && (!residual || ldr >= k) && (!hidden || ldh >= k) && (!normed || ldn >= k),
               "rms_norm_quant: leading dimension smaller than the row");
  if (m == 0) return QTTS_OK;
  QTTS_REQUIRE(sx && (k == 0 || (x && weight && qx)), "rms_norm_quant: null pointer");
  const int64_t e = dtype_size(x_dtype);
  QTTS_REQUIRE(!spans_overlap(x, m, ldx, k, e, qx, m, k, k, 1) &&
                   !(residual && spans_overlap(residual, m, ldr, k, e, qx, m, k, k, 1)),
               "rms_norm_quant: qx overlaps the activations");
  QTTS_REQUIRE(!hidden || (hidden == x && ldh == ldx) || !spans_overlap(x, m, ldx, k, e, hidden, m, ldh, k, e),
               "rms_norm_quant: hidden overlaps x");
  QTTS_REQUIRE(!hidden || !residual || (hidden == residual && ldh == ldr) ||
                   !spans_overlap(residual, m, ldr, k, e, hidden, m, ldh, k, e),
               "rms_norm_quant: hidden overlaps the residual");
  QTTS_REQUIRE(!normed || (!spans_overlap(x, m, ldx, k, e, normed, m, ldn, k, e) &&
                           !(residual && spans_overlap(residual, m, ldr, k, e, normed, m, ldn, k, e)) &&
                           !(hidden && spans_overlap(hidden, m, ldh, k, e, normed, m, ldn, k, e))),
               "rms_norm_quant: normed overlaps the activations");
  QTTS_TRY(current_device_check());
  return qtts_launch_rms_norm_quant(x, x_dtype, m, k, ldx, residual, ldr, weight, eps, codes, qx, sx, hidden, ldh, normed,
                                    ldn, (hipStream_t)stream);
}

int qtts_silu_mul_quant(const void* gate_up, int x_dtype, int64_t m, int64_t k, int64_t ld_gate_up, int codes, void* qx,
                        float* sx, void* act, int64_t ldact, void* stream) {
  QTTS_REQUIRE(m >= 0 && k >= 0, "silu_mul_quant: negative size");
  QTTS_REQUIRE(m < (1ll << 31) && k < (1ll << 30), "silu_mul_quant: size too large");
  QTTS_REQUIRE(dtype_ok(x_dtype), "silu_mul_quant: bad dtype code");
  QTTS_REQUIRE(codes == QTTS_CODE_INT8 || codes == QTTS_CODE_E4M3, "silu_mul_quant: bad code kind %d", codes);
  QTTS_REQUIRE(ld_gate_up >= 2 * k && (!act || ldact >= k), "silu_mul_quant: leading dimension smaller than the row");
  if (m == 0) return QTTS_OK;
  QTTS_REQUIRE(sx && (k == 0 || (gate_up && qx)), "silu_mul_quant: null pointer");
  const int64_t e = dtype_size(x_dtype);
  QTTS_REQUIRE(!spans_overlap(gate_up, m, ld_gate_up, 2 * k, e, qx, m, k, k, 1), "silu_mul_quant: qx overlaps gate_up");
  QTTS_REQUIRE(!act || !spans_overlap(gate_up, m, ld_gate_up, 2 * k, e, act, m, ldact, k, e),
               "silu_mul_quant: act overlaps gate_up");
  QTTS_TRY(current_device_check());
  return qtts_launch_silu_mul_quant(gate_up, x_dtype, m, k, ld_gate_up, codes, qx, sx, act, ldact, (hipStream_t)stream);
}

int64_t qtts_lora_plan_bytes(int64_t m, int64_t slots) {
  if (m < 0 || slots < 0 || m >= (1ll << 31) || slots >= (1ll << 30))
    return qtts_set_error(QTTS_ERR_INVALID_ARGUMENT, "lora_plan: bad sizes");
  return slots > qtts::kPlanMaxSlots || m > qtts::kPlanMaxRows ? 0 : qtts::plan_words(m, slots) * 4;
}

int qtts_lora_plan(const int32_t* index, int64_t m, int64_t slots, int32_t* plan, int64_t plan_bytes, void* stream) {
  const int64_t need = qtts_lora_plan_bytes(m, slots);
  if (need < 0) return (int)need;
  QTTS_REQUIRE(slots <= qtts::kPlanMaxSlots && m <= qtts::kPlanMaxRows, "lora_plan: more than %d slots or %lld rows",
               qtts::kPlanMaxSlots, (long long)qtts::kPlanMaxRows);
  QTTS_REQUIRE(plan && (uintptr_t)plan % 16 == 0 && (m == 0 || index), "lora_plan: null or unaligned pointer");
  QTTS_REQUIRE(plan_bytes >= need, "lora_plan: plan of %lld bytes < %lld needed", (long long)plan_bytes, (long long)need);
  QTTS_TRY(current_device_check());
  return qtts_launch_lora_plan(index, m, slots, plan, (hipStream_t)stream);
}

static int lora_add(const void* x, int x_dtype, int64_t m, int64_t k, int64_t ldx, const int32_t* index, const int32_t* plan,
                    int64_t slots, const void* a, const void* b, int64_t rank, const int32_t* ranks, const float* scaling,
                    const int64_t* part_ends, int64_t parts, const void* base, int64_t ldb, void* out, int64_t n, int64_t ldo,
                    bool whole, void* ws, int64_t ws_bytes, void* stream) {
  QTTS_REQUIRE(m >= 0 && n >= 0 && k >= 0 && slots >= 0, "lora_add: negative size");
  QTTS_REQUIRE(m < (1ll << 31) && n < (1ll << 30) && k < (1ll << 30) && slots < (1ll << 30), "lora_add: size too large");
  QTTS_REQUIRE(x_dtype == QTTS_BF16 || x_dtype == QTTS_F16, "lora_add: activations must be bf16 or fp16");
  QTTS_REQUIRE(rank >= 1 && rank <= QTTS_LORA_MAX_RANK, "lora_add: rank %lld is not in 1..%d", (long long)rank,
               QTTS_LORA_MAX_RANK);
  QTTS_REQUIRE(parts >= 1 && parts <= QTTS_LORA_MAX_PARTS && part_ends, "lora_add: %lld partitions are not in 1..%d",
               (long long)parts, QTTS_LORA_MAX_PARTS);
  for (int64_t p = 0; p < parts; ++p)
    QTTS_REQUIRE(part_ends[p] >= (p ? part_ends[p - 1] : 0), "lora_add: partition ends do not ascend");
  QTTS_REQUIRE(part_ends[parts - 1] == n, "lora_add: the partitions end at %lld of %lld columns",
               (long long)part_ends[parts - 1], (long long)n);
  QTTS_REQUIRE(ldx >= k && ldb >= n && ldo >= n, "lora_add: leading dimension smaller than the row");
  QTTS_REQUIRE(ws_bytes >= 0, "lora_add: negative workspace size");
  if (m == 0 || n == 0) return QTTS_OK;
  QTTS_REQUIRE((uintptr_t)plan % 16 == 0, "lora_add: unaligned plan");
  QTTS_REQUIRE(base && out && index && (slots == 0 || (scaling && b && (k == 0 || (x && a)))), "lora_add: null pointer");
  QTTS_REQUIRE((out == base && ldo == ldb) || !spans_overlap(base, m, ldb, n, 2, out, m, ldo, n, 2),
               "lora_add: out overlaps base");
  QTTS_REQUIRE(!spans_overlap(x, m, ldx, k, 2, out, m, ldo, n, 2), "lora_add: out overlaps x");
  const int64_t need = qtts_lora_ws_bytes(m, parts, rank);
  if (!ws || ws_bytes < need)
    return qtts_set_error(QTTS_ERR_WORKSPACE, "lora_add: workspace of %lld bytes < %lld needed", (long long)ws_bytes,
                          (long long)need);
  QTTS_TRY(current_device_check());
  qtts::LoraArgs g = {};
  g.x = x;
  g.ldx = ldx;
  g.index = index;
  g.plan = plan;
  g.a = a;
  g.b = b;
  g.ranks = ranks;
  g.scaling = scaling;
  g.base = base;
  g.ldb = ldb;
  g.out = out;
  g.ldo = ldo;
  g.m = m;
  g.k = (int)k;
  g.n = (int)n;
  g.slots = (int)slots;
  g.rank = (int)rank;
  g.parts.count = (int)parts;
  for (int64_t p = 0; p < parts; ++p) g.parts.end[p] = (int32_t)part_ends[p];
  g.whole = whole;
  return qtts_launch_lora_add(g, x_dtype, ws, (hipStream_t)stream);
}

int qtts_lora_add(const void* x, int x_dtype, int64_t m, int64_t k, int64_t ldx, const int32_t* index, const int32_t* plan,
                  int64_t slots, const void* a, const void* b, int64_t rank, const int32_t* ranks, const float* scaling,
                  const int64_t* part_ends, int64_t parts, const void* base, int64_t ldb, void* out, int64_t n, int64_t ldo,
                  void* ws, int64_t ws_bytes, void* stream) {
  return lora_add(x, x_dtype, m, k, ldx, index, plan, slots, a, b, rank, ranks, scaling, part_ends, parts, base, ldb, out, n,
                  ldo, false, ws, ws_bytes, stream);
}

int qtts_lora_add_fresh(const void* x, int x_dtype, int64_t m, int64_t k, int64_t ldx, const int32_t* index,
                        const int32_t* plan, int64_t slots, const void* a, const void* b, int64_t rank, const int32_t* ranks,
                        const float* scaling, const int64_t* part_ends, int64_t parts, const void* base, int64_t ldb, void* out,
                        int64_t n, int64_t ldo, void* ws, int64_t ws_bytes, void* stream) {
  return lora_add(x, x_dtype, m, k, ldx, index, plan, slots, a, b, rank, ranks, scaling, part_ends, parts, base, ldb, out, n,
                  ldo, true, ws, ws_bytes, stream);
}

int qtts_w8a16_fused_gemm_strips(const void* x, int x_dtype, int64_t m, int64_t k, int64_t ldx, int prologue,
                                 const void* norm_weight, float eps, const int8_t* qs, int64_t n, const void* scale,
                                 int scale_dtype, const void* bias, const void* residual, int64_t ldr, void* y,
                                 int64_t ldy, int algo, void* ws, int64_t ws_bytes, void* stream) {
  const qtts::WeightPolicy policy(algo);  // takes QTTS_ALGO_STREAM out of algo
  QTTS_REQUIRE(m >= 0 && n >= 0 && k >= 0, "w8a16_fused_gemm_strips: negative size");
  QTTS_REQUIRE(m < 65536 && n < (1ll << 31) && k < (1ll << 30), "w8a16_fused_gemm_strips: size too large");
  QTTS_REQUIRE(x_dtype == QTTS_BF16 || x_dtype == QTTS_F16, "w8a16_fused_gemm_strips: activations must be bf16 or fp16");
  QTTS_REQUIRE(dtype_ok(scale_dtype), "w8a16_fused_gemm_strips: bad scale dtype code");
  QTTS_REQUIRE(algo_ok_rows(algo), "w8a16_fused_gemm_strips: bad algo %d", algo);
  QTTS_REQUIRE(prologue == QTTS_PRO_NONE || prologue == QTTS_PRO_SILU_MUL || prologue == QTTS_PRO_RMS_NORM,
               "w8a16_fused_gemm_strips: bad prologue %d", prologue);
  QTTS_REQUIRE(k % 64 == 0, "w8a16_fused_gemm_strips: K %% 64 != 0 (K=%lld)", (long long)k);
  QTTS_REQUIRE(ldx >= (prologue == QTTS_PRO_SILU_MUL ? 2 * k : k) && ldy >= n && (!residual || ldr >= n),
               "w8a16_fused_gemm_strips: leading dimension smaller than the row");
  QTTS_REQUIRE(ws_bytes >= 0, "w8a16_fused_gemm_strips: negative workspace size");
  if (m == 0 || n == 0) return QTTS_OK;
  QTTS_REQUIRE(x && qs && scale && y && (prologue != QTTS_PRO_RMS_NORM || norm_weight),
               "w8a16_fused_gemm_strips: null pointer");
  QTTS_REQUIRE(prologue != QTTS_PRO_NONE || ((uintptr_t)x % 16 == 0 && (m == 1 || ldx % 8 == 0)),
               "w8a16_fused_gemm_strips: activation rows must be 16-byte aligned");
  QTTS_REQUIRE(!residual || residual == y || !ranges_overlap(residual, m, ldr, y, m, ldy, n, 2),
               "w8a16_fused_gemm_strips: residual overlaps y without being y");
  QTTS_REQUIRE(!residual || residual != y || ldr == ldy, "w8a16_fused_gemm_strips: residual is y with another stride");
  QTTS_REQUIRE(!spans_overlap(x, m, ldx, prologue == QTTS_PRO_SILU_MUL ? 2 * k : k, 2, y, m, ldy, n, 2),
               "w8a16_fused_gemm_strips: y overlaps x");
  QTTS_TRY(current_device_check());
  return qtts_launch_w8a16_fused(x, x_dtype, m, k, ldx, prologue, norm_weight, eps, qs, n, scale, scale_dtype, bias,
                                 residual, ldr, y, ldy, algo, ws, ws_bytes, (hipStream_t)stream);
}

int qtts_w8a16_gate_up_silu_strips(const void* x, int x_dtype, int64_t m, int64_t k, int64_t ldx, int prologue,
                                   const void* norm_weight, float eps, const int8_t* qs, int64_t n, const void* scale,
                                   int scale_dtype, const void* bias, void* act, int64_t ldact, int algo, void* ws,
                                   int64_t ws_bytes, void* stream) {
  const qtts::WeightPolicy policy(algo);  // takes QTTS_ALGO_STREAM out of algo
  QTTS_REQUIRE(m >= 0 && n >= 0 && k >= 0, "w8a16_gate_up_silu_strips: negative size");
  QTTS_REQUIRE(m < 65536 && n < (1ll << 31) && k < (1ll << 30), "w8a16_gate_up_silu_strips: size too large");
  QTTS_REQUIRE(x_dtype == QTTS_BF16 || x_dtype == QTTS_F16,
               "w8a16_gate_up_silu_strips: activations must be bf16 or fp16");
  QTTS_REQUIRE(dtype_ok(scale_dtype), "w8a16_gate_up_silu_strips: bad scale dtype code");
  QTTS_REQUIRE(algo_ok_rows(algo), "w8a16_gate_up_silu_strips: bad algo %d", algo);
  QTTS_REQUIRE(prologue == QTTS_PRO_NONE || prologue == QTTS_PRO_RMS_NORM,
               "w8a16_gate_up_silu_strips: prologue must be none or RMSNorm, got %d", prologue);
  QTTS_REQUIRE(k % 64 == 0, "w8a16_gate_up_silu_strips: K %% 64 != 0 (K=%lld)", (long long)k);
  QTTS_REQUIRE(n % 2 == 0, "w8a16_gate_up_silu_strips: gate_up width %lld is odd", (long long)n);
  QTTS_REQUIRE(ldx >= k && ldact >= n / 2, "w8a16_gate_up_silu_strips: leading dimension smaller than the row");
  QTTS_REQUIRE(ws_bytes >= 0, "w8a16_gate_up_silu_strips: negative workspace size");
  if (m == 0 || n == 0) return QTTS_OK;
  QTTS_REQUIRE(x && qs && scale && act && (prologue != QTTS_PRO_RMS_NORM || norm_weight),
               "w8a16_gate_up_silu_strips: null pointer");
  QTTS_REQUIRE((uintptr_t)x % 16 == 0 && (m == 1 || ldx % 8 == 0),
               "w8a16_gate_up_silu_strips: activation rows must be 16-byte aligned");
  QTTS_REQUIRE(!spans_overlap(x, m, ldx, k, 2, act, m, ldact, n / 2, 2), "w8a16_gate_up_silu_strips: act overlaps x");
  QTTS_TRY(current_device_check());
  return qtts_launch_w8a16_gate_up_silu(x, x_dtype, m, k, ldx, prologue, norm_weight, eps, qs, n, scale, scale_dtype,
                                        bias, act, ldact, algo, ws, ws_bytes, (hipStream_t)stream);
}

int qtts_fp8w_gemm_strips(const void* x, int x_dtype, int64_t m, int64_t k, int64_t ldx, const uint8_t* qs, int64_t n,
                          const float* scale, const void* bias, void* y, int64_t ldy, int algo, void* ws,
                          int64_t ws_bytes, void* stream) {
  const qtts::WeightPolicy policy(algo);  // takes QTTS_ALGO_STREAM out of algo
  QTTS_REQUIRE(m >= 0 && n >= 0 && k >= 0, "fp8w_gemm_strips: negative size (m=%lld, n=%lld, k=%lld)", (long long)m,
               (long long)n, (long long)k);
  QTTS_REQUIRE(m < (1ll << 31) && n < (1ll << 31) && k < (1ll << 31), "fp8w_gemm_strips: size too large");
  QTTS_REQUIRE(x_dtype == QTTS_BF16 || x_dtype == QTTS_F16, "fp8w_gemm_strips: activations must be bf16 or fp16");
  QTTS_REQUIRE(algo_ok(algo), "fp8w_gemm_strips: bad algo %d", algo);
  QTTS_REQUIRE(k % 64 == 0, "fp8w_gemm_strips: K %% 64 != 0 (K=%lld)", (long long)k);
  QTTS_REQUIRE(ldx >= k && ldy >= n, "fp8w_gemm_strips: leading dimension smaller than the row");
  QTTS_REQUIRE(ws_bytes >= 0, "fp8w_gemm_strips: negative workspace size");
  if (m == 0 || n == 0) return QTTS_OK;
  QTTS_REQUIRE(x && qs && scale && y, "fp8w_gemm_strips: null pointer");
  QTTS_REQUIRE((uintptr_t)x % 16 == 0 && (m == 1 || ldx % 8 == 0), "fp8w_gemm_strips: activation rows must be 16-byte aligned");
  QTTS_REQUIRE(!spans_overlap(x, m, ldx, k, 2, y, m, ldy, n, 2), "fp8w_gemm_strips: y overlaps x");
  QTTS_TRY(current_device_check());
  return qtts_launch_fp8w(x, x_dtype, m, k, ldx, qs, n, scale, bias, y, ldy, algo, ws, ws_bytes, (hipStream_t)stream);
}

int64_t qtts_strip_bytes(int64_t n, int64_t k, int kind) {
  if (n < 0 || k < 0 || n >= (1ll << 31) || k >= (1ll << 31) || (kind != QTTS_STRIP_INT8 && kind != QTTS_STRIP_FP8))
    return qtts_set_error(QTTS_ERR_INVALID_ARGUMENT, "strip_bytes: bad arguments");
  return qtts::strip_bytes(n, k, kind);
}

int qtts_to_strips(const void* src, int64_t n, int64_t k, int64_t ld_src, int kind, void* dst, void* stream) {
  QTTS_REQUIRE(n >= 0 && k >= 0 && n < (1ll << 31) && k < (1ll << 31) && ld_src >= k, "to_strips: bad sizes");
  QTTS_REQUIRE(kind == QTTS_STRIP_INT8 || kind == QTTS_STRIP_FP8, "to_strips: bad kind %d", kind);
  if (n == 0 || k == 0) return QTTS_OK;
  QTTS_REQUIRE(src && dst, "to_strips: null pointer");
  QTTS_REQUIRE((uintptr_t)dst % 16 == 0, "to_strips: destination must be 16-byte aligned");
  QTTS_TRY(current_device_check());
  return qtts_launch_to_strips(src, n, k, ld_src, dst, kind, (hipStream_t)stream);
}

int qtts_from_strips(const void* src, int64_t n, int64_t k, int kind, void* dst, int64_t ld_dst, void* stream) {
  QTTS_REQUIRE(n >= 0 && k >= 0 && n < (1ll << 31) && k < (1ll << 31) && ld_dst >= k, "from_strips: bad sizes");
  QTTS_REQUIRE(kind == QTTS_STRIP_INT8 || kind == QTTS_STRIP_FP8, "from_strips: bad kind %d", kind);
  if (n == 0 || k == 0) return QTTS_OK;
  QTTS_REQUIRE(src && dst, "from_strips: null pointer");
  QTTS_REQUIRE((uintptr_t)src % 16 == 0, "from_strips: source must be 16-byte aligned");
  QTTS_TRY(current_device_check());
  return qtts_launch_from_strips(src, n, k, dst, ld_dst, kind, (hipStream_t)stream);
}

int qtts_dequant_strips(const void* qs, int codes, int64_t n, int64_t k, const void* scale, int scale_dtype, void* w,
                        int w_dtype, int64_t ldw, void* stream) {
  QTTS_REQUIRE(n >= 0 && k >= 0 && n < (1ll << 31) && k < (1ll << 31) && ldw >= k, "dequant_strips: bad sizes");
  QTTS_REQUIRE(n < (1ll << 31) && k < (1ll << 31), "dequant_strips: size too large");
  QTTS_REQUIRE(codes == QTTS_CODE_INT8 || codes == QTTS_CODE_E4M3, "dequant_strips: bad code kind %d", codes);
  QTTS_REQUIRE(dtype_ok(scale_dtype) && dtype_ok(w_dtype), "dequant_strips: bad dtype code");
  if (n == 0 || k == 0) return QTTS_OK;
  QTTS_REQUIRE(qs && scale && w, "dequant_strips: null pointer");
  QTTS_REQUIRE((uintptr_t)qs % 16 == 0, "dequant_strips: strip buffer must be 16-byte aligned");
  QTTS_TRY(current_device_check());
  return qtts_launch_dequant_strips(qs, codes, n, k, scale, scale_dtype, w, w_dtype, ldw, (hipStream_t)stream);
}

// ---- attention over a paged cache ---------------------------------------------------------

// log2 of a page's tokens, or -1 for a size that no page has.
static int page_shift_of(int64_t page_size) {
  for (int s = qtts::kPagedMinShift; s <= qtts::kPagedMaxShift; ++s)
    if (page_size == (1ll << s)) return s;
  return -1;
}

// The checks that every call on a page table shares: sizes in 32 bits, slots and a request's capacity among them.
static int paged_sizes(const char* what, int64_t requests, int64_t cols, int64_t pages, int64_t page_size) {
  QTTS_REQUIRE(requests >= 0 && cols >= 0 && pages >= 0, "%s: negative size", what);
  QTTS_REQUIRE(page_shift_of(page_size) >= 0, "%s: a page of %lld tokens is no power of two from 16 to 1024", what,
               (long long)page_size);
  QTTS_REQUIRE(requests <= qtts::kPagedMaxRequests, "%s: %lld requests, at most %d", what, (long long)requests,
               qtts::kPagedMaxRequests);
  QTTS_REQUIRE(pages < (1ll << 31) / page_size && cols <= (1ll << 30) / page_size,
               "%s: size too large (2^31 tokens of the cache or more than 2^30 of a request)", what);
  return QTTS_OK;
}

static int paged_cache(const char* what, qtts::PagedCache& c, const void* k, const void* v, int64_t pages, int64_t page_size,
                       int64_t heads, int64_t kv_heads, int64_t d) {
  QTTS_REQUIRE(heads >= 1 && kv_heads >= 1 && heads % kv_heads == 0 && heads <= 4096,
               "%s: %lld query heads for %lld key-value heads", what, (long long)heads, (long long)kv_heads);
  QTTS_REQUIRE(d >= 16 && d <= qtts::kPagedMaxDim && d % 16 == 0, "%s: heads of %lld, not a multiple of 16 up to %d", what,
               (long long)d, qtts::kPagedMaxDim);
  QTTS_REQUIRE(pages == 0 || (k && v), "%s: null pointer", what);
  QTTS_REQUIRE(((uintptr_t)k | (uintptr_t)v) % 16 == 0, "%s: unaligned cache", what);
  c.k = const_cast<void*>(k);
  c.v = const_cast<void*>(v);
  c.pages = (int32_t)pages;
  c.page_shift = page_shift_of(page_size);
  c.kv_heads = (int32_t)kv_heads;
  c.d = (int32_t)d;
  return QTTS_OK;
}

int qtts_paged_step(const int32_t* added, int64_t requests, const int32_t* lengths, int32_t* table, int64_t cols,
                    const int32_t* free_pages, int64_t pages, const int32_t* taken, int64_t page_size, int64_t rows,
                    int64_t room, int64_t max_new, int32_t* starts, int32_t* counts, int32_t* lengths_out, int32_t* taken_out,
                    int32_t* positions, int32_t* slots, void* ws, int64_t ws_bytes, void* stream) {
  QTTS_TRY(paged_sizes("paged_step", requests, cols, pages, page_size));
  QTTS_REQUIRE(rows >= 0 && max_new >= 0, "paged_step: negative size");
  QTTS_REQUIRE(room >= rows, "paged_step: room for %lld of %lld rows", (long long)room, (long long)rows);
  QTTS_REQUIRE(room < (1ll << 31) - 8192, "paged_step: size too large");
  QTTS_REQUIRE(taken && starts && taken_out, "paged_step: null pointer");
  QTTS_REQUIRE(requests == 0 || (added && lengths && counts && lengths_out && (cols == 0 || table)), "paged_step: null pointer");
  QTTS_REQUIRE((pages == 0 || free_pages) && (room == 0 || (positions && slots)), "paged_step: null pointer");
  if (!ws || ws_bytes < qtts::kCounterBytes)
    return qtts_set_error(QTTS_ERR_WORKSPACE, "paged_step: workspace of %lld bytes < %lld needed", (long long)ws_bytes,
                          (long long)qtts::kCounterBytes);
  QTTS_TRY(current_device_check());
  qtts::PagedStepArgs a = {};
  a.added = added;
  a.lengths = lengths;
  a.table = table;
  a.free_pages = free_pages;
  a.taken = taken;
  a.starts = starts;
  a.counts = counts;
  a.lengths_out = lengths_out;
  a.taken_out = taken_out;
  a.positions = positions;
  a.slots = slots;
  a.ticket = (uint32_t*)ws;
  a.requests = (int32_t)requests;
  a.cols = (int32_t)cols;
  a.pages = (int32_t)pages;
  a.page_shift = page_shift_of(page_size);
  a.rows = (int32_t)rows;
  a.room = (int32_t)room;
  a.max_new = (int32_t)std::min<int64_t>(max_new, rows);
  return qtts_launch_paged_step(a, (hipStream_t)stream);
}

int qtts_paged_release(const int32_t* which, int64_t requests, int32_t* lengths, const int32_t* table, int64_t cols,
                       int32_t* free_pages, int64_t pages, int32_t* taken, int64_t page_size, void* stream) {
  QTTS_TRY(paged_sizes("paged_release", requests, cols, pages, page_size));
  if (requests == 0 || cols == 0 || pages == 0) return QTTS_OK;
  QTTS_REQUIRE(which && lengths && table && free_pages && taken, "paged_release: null pointer");
  QTTS_TRY(current_device_check());
  return qtts_launch_paged_release(which, lengths, table, (int)requests, (int)cols, free_pages, (int)pages, taken,
                                   page_shift_of(page_size), (hipStream_t)stream);
}

int qtts_qkv_to_cache(const void* qkv, int dtype, int64_t rows, int64_t ldqkv, int64_t heads, int64_t kv_heads, int64_t d,
                      const int32_t* positions, const int32_t* slots, const void* q_norm, const void* k_norm, float eps,
                      const float* cos, const float* sin, int64_t rope_rows, void* k, void* v, int64_t pages,
                      int64_t page_size, void* q, void* stream) {
  QTTS_TRY(paged_sizes("qkv_to_cache", 0, 0, pages, page_size));
  QTTS_REQUIRE(dtype == QTTS_BF16 || dtype == QTTS_F16, "qkv_to_cache: activations must be bf16 or fp16");
  qtts::QkvCacheArgs a = {};
  QTTS_TRY(paged_cache("qkv_to_cache", a.cache, k, v, pages, page_size, heads, kv_heads, d));
  const int64_t width = (heads + 2 * kv_heads) * d;
  QTTS_REQUIRE(rows >= 0 && rope_rows >= 0, "qkv_to_cache: negative size");
  QTTS_REQUIRE(rows < (1ll << 24) && rope_rows < (1ll << 31), "qkv_to_cache: size too large");
  QTTS_REQUIRE(ldqkv >= width, "qkv_to_cache: leading dimension smaller than the row");
  QTTS_REQUIRE(ldqkv < (1ll << 36), "qkv_to_cache: size too large");
  QTTS_REQUIRE((cos == nullptr) == (sin == nullptr) && (!cos || rope_rows > 0), "qkv_to_cache: half a rotation table");
  QTTS_REQUIRE(!(q_norm || k_norm) || (eps >= 0 && eps < INFINITY), "qkv_to_cache: an eps of %g", (double)eps);
  if (rows == 0) return QTTS_OK;
  QTTS_REQUIRE(qkv && slots && q && (!cos || positions), "qkv_to_cache: null pointer");
  QTTS_REQUIRE(((uintptr_t)qkv | (uintptr_t)q | (uintptr_t)q_norm | (uintptr_t)k_norm | (uintptr_t)cos | (uintptr_t)sin) % 16 == 0 &&
                   ldqkv % 8 == 0, "qkv_to_cache: rows, norm weights and angles must start on 16 bytes");
  QTTS_REQUIRE(!spans_overlap(qkv, rows, ldqkv, width, 2, q, rows, heads * d, heads * d, 2), "qkv_to_cache: q overlaps qkv");
  const int64_t held = pages * page_size * kv_heads * d;
  for (const void* c : {(const void*)k, (const void*)v})
    QTTS_REQUIRE(!spans_overlap(c, 1, held, held, 2, q, rows, heads * d, heads * d, 2) &&
                     !spans_overlap(c, 1, held, held, 2, qkv, rows, ldqkv, width, 2), "qkv_to_cache: the cache overlaps q or qkv");
  QTTS_TRY(current_device_check());
  a.qkv = qkv;
  a.ldqkv = ldqkv;
  a.positions = positions;
  a.slots = slots;
  a.q_norm = q_norm;
  a.k_norm = k_norm;
  a.cos = cos;
  a.sin = sin;
  a.q = q;
  a.rows = (int32_t)rows;
  a.heads = (int32_t)heads;
  a.rope_rows = (int32_t)rope_rows;
  a.eps = eps;
  return qtts_launch_qkv_to_cache(a, dtype, (hipStream_t)stream);
}

static int paged_attention(bool weights16, const void* q, int dtype, int64_t rows, int64_t ldq, int64_t heads, int64_t kv_heads,
                           int64_t d, const void* k, const void* v, int64_t pages, int64_t page_size, const int32_t* table,
                           int64_t requests, int64_t cols, const int32_t* starts, const int32_t* counts, const int32_t* lengths,
                           const int32_t* slots, int64_t min_new, int64_t max_new, int64_t window, int64_t sinks, float scale,
                           void* out, int64_t ldo, void* ws, int64_t ws_bytes, void* stream) {
  QTTS_TRY(paged_sizes("paged_attention", requests, cols, pages, page_size));
  QTTS_REQUIRE(dtype == QTTS_BF16 || dtype == QTTS_F16, "paged_attention: activations must be bf16 or fp16");
  qtts::PagedAttentionArgs a = {};
  QTTS_TRY(paged_cache("paged_attention", a.cache, k, v, pages, page_size, heads, kv_heads, d));
  QTTS_REQUIRE(rows >= 0 && min_new >= 0 && max_new >= 0 && window >= 0 && sinks >= 0, "paged_attention: negative size");
  QTTS_REQUIRE(rows < (1ll << 24) && rows * heads < (1ll << 31), "paged_attention: size too large");
  QTTS_REQUIRE(ldq >= heads * d && ldo >= heads * d, "paged_attention: leading dimension smaller than the row");
  QTTS_REQUIRE(ldq < (1ll << 36) && ldo < (1ll << 36), "paged_attention: size too large");
  // (up to where the scale of exponentials of 2 is finite)
  QTTS_REQUIRE(scale > 0 && scale <= 2e38f, "paged_attention: scale %g is not in (0, 2e38]", (double)scale);
  QTTS_REQUIRE(ws_bytes >= 0, "paged_attention: negative workspace size");
  if (rows == 0) return QTTS_OK;
  QTTS_REQUIRE(q && out && slots && (requests == 0 || (starts && counts && lengths && (cols == 0 || table))),
               "paged_attention: null pointer");
  QTTS_REQUIRE(((uintptr_t)q | (uintptr_t)out) % 16 == 0 && ldq % 8 == 0 && ldo % 8 == 0,
               "paged_attention: rows must start on 16 bytes");
  QTTS_REQUIRE(!spans_overlap(q, rows, ldq, heads * d, 2, out, rows, ldo, heads * d, 2), "paged_attention: out overlaps q");
  const int64_t held = pages * page_size * kv_heads * d;
  for (const void* c : {k, v})
    QTTS_REQUIRE(!spans_overlap(c, 1, held, held, 2, out, rows, ldo, heads * d, 2), "paged_attention: out overlaps the cache");
  const int64_t need = qtts_paged_attention_ws_bytes(std::min(max_new, rows) * (heads / kv_heads), d);
  if (!ws || ws_bytes < need)
    return qtts_set_error(QTTS_ERR_WORKSPACE, "paged_attention: workspace of %lld bytes < %lld needed", (long long)ws_bytes,
                          (long long)need);
  QTTS_TRY(current_device_check());
  a.q = q;
  a.ldq = ldq;
  a.out = out;
  a.ldo = ldo;
  a.table = table;
  a.starts = starts;
  a.counts = counts;
  a.lengths = lengths;
  a.rows = (int32_t)rows;
  a.heads = (int32_t)heads;
  a.requests = (int32_t)requests;
  a.cols = pages ? (int32_t)cols : 0;  // no pages hold no tokens
  a.max_new = (int32_t)std::min<int64_t>(max_new, rows);
  a.window = (int32_t)std::min<int64_t>(window, INT32_MAX);
  a.sinks = (int32_t)std::min<int64_t>(sinks, INT32_MAX);
  a.scale = scale * 1.44269504088896340736f;  // exponentials of 2
  a.weights16 = weights16;
  return qtts_launch_paged_attention(a, (int)std::min<int64_t>(min_new, rows), dtype, ws, (hipStream_t)stream);
}

int qtts_paged_attention(const void* q, int dtype, int64_t rows, int64_t ldq, int64_t heads, int64_t kv_heads, int64_t d,
                         const void* k, const void* v, int64_t pages, int64_t page_size, const int32_t* table, int64_t requests,
                         int64_t cols, const int32_t* starts, const int32_t* counts, const int32_t* lengths,
                         const int32_t* slots, int64_t min_new, int64_t max_new, int64_t window, int64_t sinks, float scale,
                         void* out, int64_t ldo, void* ws, int64_t ws_bytes, void* stream) {
  return paged_attention(false, q, dtype, rows, ldq, heads, kv_heads, d, k, v, pages, page_size, table, requests, cols, starts, counts,
                         lengths, slots, min_new, max_new, window, sinks, scale, out, ldo, ws, ws_bytes, stream);
}

int qtts_paged_attention_w16(const void* q, int dtype, int64_t rows, int64_t ldq, int64_t heads, int64_t kv_heads, int64_t d,
                             const void* k, const void* v, int64_t pages, int64_t page_size, const int32_t* table, int64_t requests,
                             int64_t cols, const int32_t* starts, const int32_t* counts, const int32_t* lengths,
                             const int32_t* slots, int64_t min_new, int64_t max_new, int64_t window, int64_t sinks, float scale,
                             void* out, int64_t ldo, void* ws, int64_t ws_bytes, void* stream) {
  return paged_attention(true, q, dtype, rows, ldq, heads, kv_heads, d, k, v, pages, page_size, table, requests, cols, starts, counts,
                         lengths, slots, min_new, max_new, window, sinks, scale, out, ldo, ws, ws_bytes, stream);
}

int qtts_kernel_timer_begin(int max_launches) {
  QTTS_REQUIRE(max_launches > 0 && max_launches <= (1 << 20), "kernel timer: max_launches must be in [1, 2^20]");
  std::lock_guard<std::mutex> lock(g_timer_mu);
  if (g_timer_armed.load(std::memory_order_relaxed))
    return qtts_set_error(QTTS_ERR_INVALID_ARGUMENT, "kernel timer: already armed");
  timer_release();
  g_timer_events.reserve(2 * (size_t)max_launches);
  for (int i = 0; i < 2 * max_launches; ++i) {
    hipEvent_t e = nullptr;
    hipError_t err = hipEventCreate(&e);
    if (err != hipSuccess) {
      timer_release();
      return qtts_set_error(QTTS_ERR_HIP, "kernel timer: hipEventCreate failed: %s", hipGetErrorString(err));
    }
    g_timer_events.push_back(e);
  }
  g_timer_untimed = 0;
  g_timer_armed.store(true, std::memory_order_release);
  return QTTS_OK;
}

int qtts_kernel_timer_end(double* total_ms, int64_t* launches, int64_t* untimed) {
  QTTS_REQUIRE(total_ms && launches && untimed, "kernel timer: null pointer");
  std::lock_guard<std::mutex> lock(g_timer_mu);
  if (!g_timer_armed.load(std::memory_order_relaxed))
    return qtts_set_error(QTTS_ERR_INVALID_ARGUMENT, "kernel timer: not armed");
  g_timer_armed.store(false, std::memory_order_release);
  double sum = 0.0;
  int status = QTTS_OK;
  for (size_t i = 0; i + 1 < g_timer_used; i += 2) {
    float ms = 0.0f;
    hipError_t err = hipEventSynchronize(g_timer_events[i + 1]);
    if (err == hipSuccess) err = hipEventElapsedTime(&ms, g_timer_events[i], g_timer_events[i + 1]);
    if (err != hipSuccess) {
      status = qtts_set_error(QTTS_ERR_HIP, "kernel timer: %s", hipGetErrorString(err));
      break;
    }
    sum += ms;
  }
  *total_ms = sum;
  *launches = (int64_t)(g_timer_used / 2);
  *untimed = g_timer_untimed;
  timer_release();
  return status;
}

}  // extern "C"
