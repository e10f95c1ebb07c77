// Attention of many rows a request over a paged cache (prompts, chunks of prompts behind cached tokens): bound by the
// matrix cores.
//
// The mathematics: S^T = K Q^T and O^T = V^T P^T with 32x32x16 MFMAs; a wave has 32 rows (a token's query heads of one
// key-value head follow each other) as its columns, 64 keys a step, running maximum and sum per column.  The keys are dealt
// to the rows of the S^T products so that the scores a lane receives are runs of eight keys, its operand of the second
// product: P never leaves its lane.  The four waves of a workgroup share the tile's keys and values in LDS, which are
// loaded there directly, one tile ahead; pieces of 16 bytes are placed so that the operand reads meet no bank twice
// (swizzles below; ds_read_b128 serves the lanes as pipe.h says).
//
// P goes to the second product in two 16-bit parts, whose products add up to P's in 16 bits (bf16) or 22 (fp16), so that sums that
// cancel keep their bits; where fp16's parts end, and what keeps a long tail above that: paged_attn.h.  In one part (W16, where the
// caller asks for it) a weight is rounded by half a step of the type: two products of three, half of the softmax's instructions.
//
// One prompt of 8192 tokens, 16 query and 8 key-value heads of 128 in bf16 (275 GFLOP): 398 us, 691 TFLOP/s (W16: 280 us, 980), where
// a large library product reaches 1530 (2250 on zeros: the card's power bounds its clock, 2.0 GHz here).  The matrix cores are
// busy 49% of the cycles and the vector units 44%, 8.3e7 instructions to 1.27e7 MFMAs (W16: 46, 41, 5.1e7, 8.5e6); LDS reads meet
// no bank twice.  With W16 it takes 252 us without the softmax, 241 without the loads, 224 without the second product: no one of
// them is what is waited for, the two waves a SIMD do not fill each other's gaps.  Operands further ahead, wave
// priorities and loads that the compiler does not count gave nothing; waves of 64 rows, one a SIMD, 373 us; the next tile's
// scores beside this one's softmax in a wave spilled 63 registers (554 us).  Both parts' products by groups of operands instead of
// one after the other: 396 us.  16384 tokens under a window of 1024: 223 us, 598 TFLOP/s of what the rows see (W16: 177, 755; every
// run of 64 tokens has two or three masked tiles of 18); 4 x 1003 tokens behind 2500 on pages of 32: 136 us, 512 (W16: 105, 660).
#include "paged_attn.h"
#include "pipe.h"

namespace qtts {

namespace {

constexpr int kTile = 64, kRun = 128, kWaves = 4, kThreads = 64 * kWaves, kWaveRows = kRun / kWaves;

typedef __attribute__((ext_vector_type(16))) float f32x16_t;

template <typename T> struct mfma32;
template <> struct mfma32<bf16_t> {
  static __device__ __forceinline__ f32x16_t mma(i32x4_t a, i32x4_t b, f32x16_t c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b), c, 0, 0, 0);
  }
};
template <> struct mfma32<f16_t> {
  static __device__ __forceinline__ f32x16_t mma(i32x4_t a, i32x4_t b, f32x16_t c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8_t, a), __builtin_bit_cast(f16x8_t, b), c, 0, 0, 0);
  }
};

// sum + lo + hi of two packed values, in one dot product with ones: where the second product takes weights of 16 bits, their sum
// is of those.
template <typename T> __device__ __forceinline__ float add2(uint32_t two, float sum) {
  typedef __attribute__((ext_vector_type(2))) _Float16 f16x2_t;
  if constexpr (std::is_same<T, bf16_t>::value)
    return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2_t, two), __builtin_bit_cast(bf16x2_t, 0x3f803f80u), sum, false);
  else
    return __builtin_amdgcn_fdot2(__builtin_bit_cast(f16x2_t, two), __builtin_bit_cast(f16x2_t, 0x3c003c00u), sum, false);
}

// Position of piece `piece` in row `row`: rows of 128 bytes two to a bank cycle, longer ones one.
template <int BYTES> __device__ __forceinline__ int place(int row, int piece) {
  return BYTES == 128 ? piece ^ ((row >> 1) & 7) : piece ^ (row & 15);
}

// The key (of 64) whose scores are row `row` of the S^T products: a lane's rows 8 b + 4 h + c are keys 16 (b / 2) + 8 h + 4 (b % 2) + c.
__device__ __forceinline__ int key_of_row(int row) {
  const int b = (row >> 3) & 3, h = (row >> 2) & 1, c = row & 3;
  return (row & 32) + 16 * (b >> 1) + 8 * h + 4 * (b & 1) + c;
}

// DP: the head size (EXACT) or what it is rounded up to, 64, 128 or 256.  WIDE: pages of a tile or more.  W16: weights of 16 bits.
template <typename T, int DP, bool EXACT, bool WIDE, bool W16> __global__ __launch_bounds__(kThreads, DP <= 128 ? 2 : 1) void paged_many_kernel(PagedLaunch p) {
  constexpr int NS = DP / 16, NB = DP / 32, KI = DP / 32;  // steps of Q K^T, blocks of O^T, 1 KiB loads a wave and operand
  __shared__ __attribute__((aligned(16))) uint8_t keys[2][kTile * DP * 2], values[2][kTile * DP * 2];
  __shared__ unsigned flag;
  const PagedAttentionArgs& a = p.a;
  const int kv_heads = a.cache.kv_heads, h = blockIdx.x % kv_heads, item = blockIdx.x / kv_heads;
  if (item >= p.items) {
    fill_rows<T>(p, blockIdx.x - p.items * kv_heads);
    return;
  }
  PagedWork w;
  if (!paged_work<kRun, kTile>(p, item, w)) return;
  const int group = a.heads / kv_heads, d = EXACT ? DP : a.cache.d, shift = a.cache.page_shift;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, col = lane & 31, half = lane >> 5;
  const int64_t rows = (int64_t)w.count * group, first_row = (int64_t)w.run * kRun;

  // tokens of the run, and of this wave's rows
  const int run_lo = w.position + (int)(first_row / group);
  const int run_hi = w.position + (int)((min(first_row + kRun, rows) - 1) / group);
  const int64_t wave_row = first_row + wave * kWaveRows;
  const bool busy = wave_row < rows;
  const int wave_lo = w.position + (int)(wave_row / group);
  const int wave_hi = busy ? w.position + (int)((min(wave_row + kWaveRows, rows) - 1) / group) : -1;

  const KeyTiles tiles = key_tiles<kTile>(run_lo, run_hi, a.window, a.sinks);
  const int splits = (tiles.count + w.chunk - 1) / w.chunk;  // w.splits or fewer
  if (w.split >= splits) return;
  const int begin = w.split * w.chunk, end = min(tiles.count, begin + w.chunk);

  const bool live = wave_row + col < rows;
  const int token = live ? (int)((wave_row + col) / group) : 0;
  const int query = h * group + (live ? (int)(wave_row + col - (int64_t)token * group) : 0);
  const int hi = live ? w.position + token : -1, lo = a.window && live ? max(0, hi - a.window + 1) : 0;
  const int wave_all_lo = a.window ? max(0, wave_hi - a.window + 1) : 0;  // every row of the wave sees [wave_all_lo, wave_lo]
  const int any_lo = a.window ? max(0, wave_lo - a.window + 1) : 0;       // and none what is below any_lo and no sink

  i32x4_t qf[NS];
  {
    const T* q = (const T*)a.q + (int64_t)(w.row + token) * a.ldq + (int64_t)query * d + half * 8;
    const i32x4_t zero = {0, 0, 0, 0};
#pragma unroll
    for (int s = 0; s < NS; ++s) qf[s] = live && s * 16 < d ? *(const i32x4_t*)(q + s * 16) : zero;
  }

  // ---- the tile's way to LDS
  const int32_t* table = a.table + (int64_t)w.request * a.cols;
  const int last = w.length - 1, mask = (1 << shift) - 1;
  const uint8_t *cache_k = (const uint8_t*)a.cache.k, *cache_v = (const uint8_t*)a.cache.v;
  auto tile_of = [&](int i) { return key_tile(tiles, min(i, end - 1)) * kTile; };
  auto head_of = [&](int32_t page) {  // bytes
    return ((int64_t)paged_page(page, a.cache.pages) * kv_heads + h) * ((int64_t)d << (shift + 1));
  };
  // the page of this lane's key of the tile (all of them on one page where pages are wide)
  auto pages_of = [&](int base) { return table[min(WIDE ? base : base + lane, last) >> shift]; };
  if constexpr (!EXACT) {  // the columns of a key past its d are zero in both buffers and stay so
    for (int i = threadIdx.x; i < 2 * kTile * DP / 8; i += kThreads) {
      const i32x4_t zero = {0, 0, 0, 0};
      *(i32x4_t*)(&keys[0][0] + 16 * i) = zero;
    }
    __syncthreads();
  }
  // Load n of this wave: units of 16 bytes (wave KI + n) 64 + lane, of keys' rows and of values' dimensions.  Its keys are of one
  // page of 16 tokens or more; its values' keys are this lane's piece of n's parity.
  auto unit_of = [&](int n) { return (wave * KI + n) * 64 + lane; };
  auto piece_of = [&](int n) { return place<DP * 2>(unit_of(n) / (DP / 8), unit_of(n) % (DP / 8)); };
  uint32_t k_at[KI], v_at[KI];  // bytes from the tile's place on its page, or from a load's page where pages are narrow
#pragma unroll
  for (int n = 0; n < KI; ++n) {
    const int key = key_of_row(unit_of(n) / (DP / 8)), dim = unit_of(n) / 8, run = place<128>(dim, unit_of(n) % 8);
    k_at[n] = (uint32_t)((WIDE ? key : key & mask) * d + piece_of(n) * 8) * 2;
    v_at[n] = ((uint32_t)min(dim, d - 1) << (shift + 1)) + (WIDE ? run * 8 : (run * 8) & mask) * 2;
  }
  auto stage = [&](int base, int32_t page, int buffer) {
    uint8_t *kb = keys[buffer] + wave * KI * 1024, *vb = values[buffer] + wave * KI * 1024;
    auto load_k = [&](const uint8_t* k, int n) {
      if (EXACT || piece_of(n) * 8 < d) load_to_lds16(k + k_at[n], kb + n * 1024);
    };
    if constexpr (WIDE) {
      const int64_t at = head_of(__builtin_amdgcn_readfirstlane(page));
      const uint8_t *k = cache_k + at + (int64_t)(base & mask) * d * 2, *v = cache_v + at + (base & mask) * 2;
#pragma unroll
      for (int n = 0; n < KI; ++n) load_k(k, n);
#pragma unroll
      for (int n = 0; n < KI; ++n) load_to_lds16(v + v_at[n], vb + n * 1024);
    } else {
#pragma unroll
      for (int n = 0; n < KI; ++n)
        load_k(cache_k + head_of(__builtin_amdgcn_readlane(page, key_of_row((wave * KI + n) * 64 / (DP / 8)))), n);
      const uint8_t* v[2];
#pragma unroll
      for (int n = 0; n < 2; ++n) v[n] = cache_v + head_of(__shfl(page, place<128>(unit_of(n) / 8, lane % 8) * 8, 64));
#pragma unroll
      for (int n = 0; n < KI; ++n) load_to_lds16(v[n & 1] + v_at[n], vb + n * 1024);
    }
  };

  f32x16_t o[NB];
  Reference<T> ref;
  float l = 0.0f;
#pragma unroll
  for (int b = 0; b < NB; ++b)
#pragma unroll
    for (int e = 0; e < 16; ++e) o[b][e] = 0.0f;

  // One tile in LDS.
  auto tile = [&](int here, const uint8_t* kb, const uint8_t* vb) {
    // Operands leave LDS some products before theirs: the barriers keep the compiler from gathering loads and uses.
    f32x16_t s[2];
    constexpr int KP = 2;
    i32x4_t k[KP][2];
    auto load_k = [&](int n) {
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const int row = t * 32 + col;
        k[n % KP][t] = *(const i32x4_t*)(kb + row * DP * 2 + place<DP * 2>(row, 2 * n + half) * 16);
      }
    };
#pragma unroll
    for (int n = 0; n < KP - 1; ++n) load_k(n);
#pragma unroll
    for (int n = 0; n < NS; ++n) {
      if (n + KP - 1 < NS) load_k(n + KP - 1);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        if (n) s[t] = mfma32<T>::mma(k[n % KP][t], qf[n], s[t]);
        else s[t] = mfma32<T>::mma(k[n % KP][t], qf[n], f32x16_t{});
      }
    }
    constexpr int VP = 4;  // values' operands that are out together; operand n: keys 16 (n / NB), columns 32 (n % NB)
    i32x4_t v[VP];
    auto load_v = [&](int n) {
      const int dim = n % NB * 32 + col;
      v[n % VP] = *(const i32x4_t*)(vb + dim * 128 + place<128>(dim, 2 * (n / NB) + half) * 16);
    };
#pragma unroll
    for (int n = 0; n < VP; ++n) load_v(n);
    __builtin_amdgcn_sched_barrier(0);
    // Score e of product t: key here + 32 t + 16 (e / 8) + 8 half + e % 8.  Where some row does not see some key of the tile: a
    // bit a key, set for those that this lane's row sees, makes each score's upper bound (infinite, or -infinite).
    if (here + kTile - 1 > wave_lo || (here < wave_all_lo && here + kTile > a.sinks)) {
      auto below = [&](int n) { return n <= 0 ? 0ull : n >= 64 ? ~0ull : (1ull << n) - 1; };  // keys here .. here + n - 1
      const uint64_t seen = (below(hi + 1 - here) & (~below(lo - here) | below(a.sinks - here))) >> (8 * half);
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const uint32_t hidden = ~(uint32_t)(seen >> (32 * t));
          const uint32_t sign = (hidden << (31 - 16 * (e >> 3) - (e & 7))) & 0x80000000u;
          s[t][e] = fminf(s[t][e], __uint_as_float(sign | 0x7f800000u));
        }
    }
    float top = s[0][0];
#pragma unroll
    for (int e = 1; e < 32; ++e) top = fmaxf(top, s[e >> 4][e & 15]);
    top = max_32(top);
    const bool now = ref.moves(top, a.scale);
    if (__any(now)) {
      const float keep = ref.move(now, top, a.scale);
      l *= keep;
#pragma unroll
      for (int b = 0; b < NB; ++b) o[b] *= keep;
    }
    if (ref.far) {
      const float off = fmaxf(ref.r, kLowest);
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int e = 0; e < 16; ++e) s[t][e] -= off;
    }
    const float add = ref.far ? kAim<T> : ref.bias;
#pragma unroll
    for (int ks = 0; ks < 4; ++ks) {
      i32x4_t p1, p2;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float w0 = exp2_hw(__builtin_fmaf(s[ks >> 1][8 * (ks & 1) + 2 * j], a.scale, add));
        const float w1 = exp2_hw(__builtin_fmaf(s[ks >> 1][8 * (ks & 1) + 2 * j + 1], a.scale, add));
        const uint32_t two = pack2<T>(w0, w1);
        p1[j] = (int)two;
        if constexpr (W16) {
          l = add2<T>(two, l);
        } else {
          l += w0 + w1;
          p2[j] = (int)pack2<T>(w0 - to_f32(T{(uint16_t)two}), w1 - to_f32(T{(uint16_t)(two >> 16)}));
        }
      }
#pragma unroll
      for (int b = 0; b < NB; ++b) {
        const int n = ks * NB + b;
        o[b] = mfma32<T>::mma(v[n % VP], p1, o[b]);
        if constexpr (!W16) o[b] = mfma32<T>::mma(v[n % VP], p2, o[b]);
        if (n + VP < 4 * NB) load_v(n + VP);
      }
    }
  };

  int base = tile_of(begin), next = tile_of(begin + 1);
  stage(base, pages_of(base), 0);
  int32_t page = pages_of(next);
  for (int i = begin; i < end; ++i) {
    const int buffer = (i - begin) & 1, here = base;
    wait_vmcnt<0>();   // this wave's share of the tile is in LDS
    barrier_only();    // everyone's is, and the other buffer's readers are done
    if (i + 1 < end) {
      stage(next, page, buffer ^ 1);
      base = next;
      next = tile_of(i + 2);
      page = pages_of(next);
    }
    if (here + kTile > w.length) {  // values behind the request's end were never written: zero
      for (int u = threadIdx.x; u < DP * 8; u += kThreads) {
        const int past = w.length - here - 8 * place<128>(u / 8, u % 8);  // values of the piece that are the request's
        i32x4_t* piece = (i32x4_t*)(values[buffer] + 16 * u);
        if (past < 8) {
          i32x4_t kept = *piece;
#pragma unroll
          for (int j = 0; j < 4; ++j) kept[j] &= past <= 2 * j ? 0 : past == 2 * j + 1 ? 0xffff : -1;
          *piece = kept;
        }
      }
      wait_lgkmcnt0();
      barrier_only();
    }
    if (here > wave_hi || (here + kTile <= any_lo && here >= a.sinks)) continue;  // out of the wave's sight
    tile(here, keys[buffer], values[buffer]);
  }
  l = sum_32(l);
  ref.r = fmaxf(ref.r, kLowest);

  // rows whose sums are not finite though their weights are, one by one
  bool odd = false;
#pragma unroll
  for (int b = 0; b < NB; ++b)
#pragma unroll
    for (int e = 0; e < 16; ++e) odd |= b * 32 + 2 * (e & ~3) < d && !(fabsf(o[b][e]) <= -kLowest);
  uint64_t again = __ballot(odd && live && l <= -kLowest);
  again = (again | (again >> 32)) & 0xffffffff;
  if (__syncthreads_or(again != 0)) {  // the tiles in LDS are done with
    float* dst = (float*)keys[0] + wave * DP;
    while (again) {
      const int n = __builtin_ctzll(again);
      again &= again - 1;
      row_again<T, kTile>(a, w, tiles, begin, 1, end, h, w.row + __builtin_amdgcn_readlane(token, n),
                          __builtin_amdgcn_readlane(query, n), __builtin_amdgcn_readlane(hi, n), __shfl(ref.r, n, 64), dst);
      wave_lds_fence();
#pragma unroll
      for (int b = 0; b < NB; ++b)
#pragma unroll
        for (int e = 0; e < 16; ++e)
          if (col == n && b * 32 + 2 * (e & ~3) < d) o[b][e] = dst[b * 32 + 2 * (e & ~3) + 4 * half + (e & 3)];
      wave_lds_fence();
    }
  }

  // element e of block b: dimension 32 b + 8 (e / 4) + 4 half + e % 4 of this lane's row
  auto put = [&](float inv) {
    T* out = (T*)a.out + (int64_t)(w.row + token) * a.ldo + (int64_t)query * d + 4 * half;
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
      for (int e = 0; e < 16; e += 4)
        if (live && b * 32 + 2 * e < d)
          *(uint64_t*)(out + b * 32 + 2 * e) = (uint64_t)pack2<T>(o[b][e] * inv, o[b][e + 1] * inv) |
                                               ((uint64_t)pack2<T>(o[b][e + 2] * inv, o[b][e + 3] * inv) << 32);
  };
  if (splits == 1) {
    put(1.0f / l);
    return;
  }
  // A part: d / 4 pairs of sums a thread, pair j of thread t at j kThreads + t, so that a wave's accesses are whole lines, then
  // [kRun] pairs of reference and weight sum.
  float* parts = p.parts + ((int64_t)w.slot * kv_heads + h) * p.slot_floats;
  const int64_t pitch = (int64_t)kv_heads * p.slot_floats;
  const int row = wave * kWaveRows + col;
  if (live) {
    float* mine = parts + w.split * pitch + 2 * threadIdx.x;
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
      for (int e = 0; e < 16; e += 2)
        if (b * 32 + 2 * (e & ~3) < d) store_pair(mine + (8 * b + e / 2) * 2 * kThreads, o[b][e], o[b][e + 1]);
    if (half == 0) store_pair(parts + w.split * pitch + kRun * d + 2 * row, ref.r, l);
  }
  wait_vmem();
  __syncthreads();
  unsigned* counter = p.counters + (int64_t)w.slot * kv_heads + h;
  if (threadIdx.x == 0) flag = __hip_atomic_fetch_add(counter, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  __syncthreads();
  if (flag != (unsigned)(splits - 1)) return;
  if (threadIdx.x == 0) reset_counter(counter);
  if (!live) return;
  float r = kLowest;
  l = 0.0f;
#pragma unroll
  for (int b = 0; b < NB; ++b)
#pragma unroll
    for (int e = 0; e < 16; ++e) o[b][e] = 0.0f;
  for (int s = 0; s < splits; ++s) {
    const float* src = parts + s * pitch;
    const f32x2_t rl = load_pair(src + kRun * d + 2 * row);
    const float now = fmaxf(r, rl[0]), keep = exp2_hw(reach_of(r, now, a.scale)), f = exp2_hw(reach_of(rl[0], now, a.scale));
    r = now;
    l = l * keep + f * rl[1];
    src += 2 * threadIdx.x;
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
      for (int e = 0; e < 16; e += 2)
        if (b * 32 + 2 * (e & ~3) < d) {
          const f32x2_t v = load_pair(src + (8 * b + e / 2) * 2 * kThreads);
          o[b][e] = o[b][e] * keep + f * v[0];
          o[b][e + 1] = o[b][e + 1] * keep + f * v[1];
        }
  }
  put(1.0f / l);
}

}  // namespace

}  // namespace qtts

int qtts_launch_paged_many(const qtts::PagedLaunch& p, int dtype, hipStream_t st) {
  using namespace qtts;
  const dim3 grid((uint32_t)((int64_t)p.items * p.a.cache.kv_heads + p.fill));
  auto go = [&](auto type, auto wide, auto w16) {
    typedef decltype(type) T;
    constexpr bool W = decltype(wide)::value, H = decltype(w16)::value;
    const int d = p.a.cache.d;
    if (d == 64) launch(paged_many_kernel<T, 64, true, W, H>, grid, dim3(kThreads), 0u, st, p);
    else if (d == 128) launch(paged_many_kernel<T, 128, true, W, H>, grid, dim3(kThreads), 0u, st, p);
    else if (d == 256) launch(paged_many_kernel<T, 256, true, W, H>, grid, dim3(kThreads), 0u, st, p);
    else if (d < 64) launch(paged_many_kernel<T, 64, false, W, H>, grid, dim3(kThreads), 0u, st, p);
    else if (d < 128) launch(paged_many_kernel<T, 128, false, W, H>, grid, dim3(kThreads), 0u, st, p);
    else launch(paged_many_kernel<T, 256, false, W, H>, grid, dim3(kThreads), 0u, st, p);
  };
  auto weights = [&](auto type, auto wide) {
    if (p.a.weights16) go(type, wide, std::true_type{});
    else go(type, wide, std::false_type{});
  };
  auto pages = [&](auto type) {
    if ((1 << p.a.cache.page_shift) >= kTile) weights(type, std::true_type{});
    else weights(type, std::false_type{});
  };
  if (dtype == QTTS_BF16) pages(bf16_t{});
  else pages(f16_t{});
  return qtts_check_launch("paged_attention");
}
