// Attention of few rows a request over a paged cache (single tokens; a count times the query heads of a key-value head up
// to 16): bound by the cache's bytes.
//
// The mathematics: S^T = K Q^T and O^T = V^T P^T with 16x16x32 MFMAs, 32 keys a wave and step, the running maximum and sum
// of the softmax per column (a row of Q).  The tile's keys are dealt to the rows of the two S^T products so that the eight
// scores that a lane receives are those of eight consecutive keys, which are the lane's operand of the second product: P
// never leaves its lane, and the values, d-major on their page, are 16-byte loads of that operand's other side.  Keys and
// values go from memory to registers and nowhere else; LDS joins the four waves at the end.
//
// P goes to the second product in two 16-bit parts, whose products add up to P's in 16 bits (bf16) or 22 (fp16): the matrix cores
// have the time (a wave's step at d = 128 is 24 MFMAs to 16 KiB of cache), and sums that cancel keep their bits.  Where fp16's
// parts end, and what keeps a long tail above that: paged_attn.h.
//
// Splits: the tiles of all requests are cut into pieces of one size, and a request's last workgroup to finish joins its
// pieces (paged_attn.h).
//
// The cache's bytes bound it: 64 requests of up to 8192 tokens, 16 query and 8 key-value heads of 128 in fp16 (1.20 GB): 222 us,
// 5.4 TB/s, as fast as the card reads (a sum over a large tensor: 5.2); one request of 65536 tokens (268 MB): 47 us,
// 5.7 TB/s with part of it left in the Infinity Cache; 27 windows of 512 tokens on pages of 16 (57 MB): 15 us, 18
// where the pages come from memory.  Short
// ones are latency: 1 x 300 tokens 9.9 us captured, of which the empty launch 2.5, the work list 1.2, the page table 1.3,
// the first tile's keys and values 3.6 and the join of the waves and splits 1.3.  Three workgroups a compute unit with
// a tile's keys and values in registers ahead of their use keep the loads out; 64 keys a step or 8 waves gave nothing.
#include "paged_attn.h"

namespace qtts {

namespace {

constexpr int kTile = 32, kRows = 16, kWaves = 4, kThreads = 64 * kWaves;

// DP: the head size (EXACT) or what it is rounded up to, 64, 128 or 256.
template <typename T, int DP, bool EXACT>
__global__ __launch_bounds__(kThreads, DP == 64 || (DP == 128 && EXACT) ? 3 : DP == 128 ? 2 : 1)
void paged_small_kernel(PagedLaunch p) {
  typedef typename mfma16<T>::vec vec;
  constexpr int NC = DP / 32, NB = DP / 16;
  __shared__ float part[kWaves][kRows][DP + 4];
  __shared__ float part_r[kWaves][kRows], part_l[kWaves][kRows];
  __shared__ unsigned flag;
  const PagedAttentionArgs& a = p.a;
  const int kv_heads = a.cache.kv_heads, h = blockIdx.x % kv_heads, item = blockIdx.x / kv_heads;
  if (item >= p.items) {
    fill_rows<T>(p, blockIdx.x - p.items * kv_heads);
    return;
  }
  PagedWork w;
  if (!paged_work<kRows, kTile>(p, item, w)) return;
  const int group = a.heads / kv_heads, d = EXACT ? DP : a.cache.d, shift = a.cache.page_shift;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, col = lane & 15, g = lane >> 4;
  const int rows = w.count * group;

  const KeyTiles tiles = key_tiles<kTile>(w.position, w.length - 1, a.window, a.sinks);
  const int begin = w.split * w.chunk, end = min(tiles.count, begin + w.chunk);
  const int splits = (tiles.count + w.chunk - 1) / w.chunk;  // w.splits or fewer
  if (w.split >= splits) return;

  // this lane's column: row `col` of the run
  const int token = col / group, query = h * group + col - token * group;
  const bool live = col < rows;
  const int hi = live ? w.position + token : -1, lo = a.window && live ? max(0, hi - a.window + 1) : 0;
  const int32_t all_lo = a.window ? max(0, w.length - a.window) : 0;  // every row sees [all_lo, w.position]
  const int32_t any_lo = a.window ? max(0, w.position - a.window + 1) : 0;  // and no row what is below any_lo and no sink
  vec qf[NC];
  {
    const T* q = (const T*)a.q + (int64_t)(w.row + (live ? token : 0)) * a.ldq + (int64_t)(live ? query : 0) * d;
    const i32x4_t zero = {0, 0, 0, 0};
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      const int dim = c * 32 + g * 8;
      qf[c] = __builtin_bit_cast(vec, live && dim < d ? *(const i32x4_t*)(q + dim) : zero);
    }
  }

  f32x4_t o[NB];
#pragma unroll
  for (int b = 0; b < NB; ++b) o[b] = f32x4_t{0, 0, 0, 0};
  Reference<T> ref;
  float l = 0.0f;

  // Key of product t's row r: base + 8 (r / 4) + 4 t + r % 4; this lane's eight scores: keys base + 8 g + 0..7.
  const int32_t* table = a.table + (int64_t)w.request * a.cols;
  const int last = (w.length - 1) & ~7, mask = (1 << shift) - 1;
  const int kgroup = (col >> 2) * 8, kin = col & 3;
  auto tile_of = [&](int i) { return key_tile(tiles, min(i, end - 1)) * kTile; };
  auto page_of = [&](int key) { return table[min(key, last) >> shift]; };
  auto head_of = [&](int32_t page) {
    return ((int64_t)paged_page(page, a.cache.pages) * kv_heads + h) * ((int64_t)d << shift);
  };
  i32x4_t kf[2][NC], vf[NB];
  auto load_k = [&](int base, int32_t page) {
    const T* k = (const T*)a.cache.k + head_of(page) + (int64_t)((min(base + kgroup, last) & mask) + kin) * d + g * 8;
    const i32x4_t zero = {0, 0, 0, 0};
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int c = 0; c < NC; ++c)
        kf[t][c] = EXACT || c * 32 + g * 8 < d ? *(const i32x4_t*)(k + (int64_t)t * 4 * d + c * 32) : zero;
  };
  auto load_v = [&](int base, int32_t page) {
    const T* v = (const T*)a.cache.v + head_of(page) + (min(base + g * 8, last) & mask) + ((int64_t)col << shift);
#pragma unroll
    for (int b = 0; b < NB; ++b) vf[b] = *(const i32x4_t*)(v + ((int64_t)(EXACT ? b : min(b, d / 16 - 1)) << (shift + 4)));
  };

  int i = begin + wave;
  if (i < end) {
    int base = tile_of(i), next = tile_of(i + kWaves);
    load_k(base, page_of(base + kgroup));
    load_v(base, page_of(base + g * 8));
    int32_t page_k = page_of(next + kgroup), page_v = page_of(next + g * 8);
    for (; i < end; i += kWaves) {
      f32x4_t s[2] = {{0, 0, 0, 0}, {0, 0, 0, 0}};
#pragma unroll
      for (int c = 0; c < NC; ++c)
#pragma unroll
        for (int t = 0; t < 2; ++t) s[t] = mfma16<T>::mma(__builtin_bit_cast(vec, kf[t][c]), qf[c], s[t]);
      const bool more = i + kWaves < end;
      if (more) load_k(next, page_k);
      const int key = base + g * 8;
      // a tile that every row sees whole needs no mask
      const bool whole = base + kTile - 1 <= w.position && (base >= all_lo || base + kTile <= a.sinks);
      float x[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) x[j] = s[j >> 2][j & 3];
      if (!whole) {
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] = key + j <= hi && (key + j >= lo || key + j < a.sinks) ? x[j] : -INFINITY;
      }
      float top = x[0];
#pragma unroll
      for (int j = 1; j < 8; ++j) top = fmaxf(top, x[j]);
      top = max_16_32(top);
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
        for (int j = 0; j < 8; ++j) x[j] -= off;
      }
      const float add = ref.far ? kAim<T> : ref.bias;
      i32x4_t p1, p2;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float w0 = exp2_hw(__builtin_fmaf(x[2 * j], a.scale, add)), w1 = exp2_hw(__builtin_fmaf(x[2 * j + 1], a.scale, add));
        l += w0 + w1;
        const uint32_t two = pack2<T>(w0, w1);
        p1[j] = (int)two;
        p2[j] = (int)pack2<T>(w0 - to_f32(T{(uint16_t)two}), w1 - to_f32(T{(uint16_t)(two >> 16)}));
      }
      if (!whole) {  // values that no row sees, among them what lies behind the request's end and was never written: zero
        uint32_t keep[4] = {0, 0, 0, 0};
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (key + j < w.length && (key + j >= any_lo || key + j < a.sinks)) keep[j >> 1] |= 0xffffu << (16 * (j & 1));
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
          for (int j = 0; j < 4; ++j) vf[b][j] = (int)((uint32_t)vf[b][j] & keep[j]);
      }
#pragma unroll
      for (int b = 0; b < NB; ++b) {
        o[b] = mfma16<T>::mma(__builtin_bit_cast(vec, vf[b]), __builtin_bit_cast(vec, p1), o[b]);
        o[b] = mfma16<T>::mma(__builtin_bit_cast(vec, vf[b]), __builtin_bit_cast(vec, p2), o[b]);
      }
      if (more) {
        load_v(next, page_v);
        base = next;
        next = tile_of(i + 2 * kWaves);
        page_k = page_of(next + kgroup);
        page_v = page_of(next + g * 8);
      }
    }
  }

  // rows whose sums are not finite though their weights are, one by one
  l = sum_16_32(l);
  ref.r = fmaxf(ref.r, kLowest);
  bool odd = false;
#pragma unroll
  for (int b = 0; b < NB; ++b)
#pragma unroll
    for (int e = 0; e < 4; ++e) odd |= b * 16 < d && !(fabsf(o[b][e]) <= -kLowest);
  uint64_t again = __ballot(odd && live && l <= -kLowest);
  again = (again | (again >> 16) | (again >> 32) | (again >> 48)) & 0xffff;
  while (again) {
    const int n = __builtin_ctzll(again);
    again &= again - 1;
    const int t = n / group;
    row_again<T, kTile>(a, w, tiles, begin + wave, kWaves, end, h, w.row + t, h * group + n - t * group, w.position + t,
                        __shfl(ref.r, n, 64), &part[wave][0][0]);
    wave_lds_fence();
#pragma unroll
    for (int b = 0; b < NB; ++b)
      if (col == n && b * 16 < d) o[b] = *(const f32x4_t*)(&part[wave][0][0] + b * 16 + g * 4);
    wave_lds_fence();
  }

  // the waves' results
  if (live) {
    if (g == 0) {
      part_r[wave][col] = ref.r;
      part_l[wave][col] = l;
    }
#pragma unroll
    for (int b = 0; b < NB; ++b)
      if (b * 16 < d) *(f32x4_t*)&part[wave][col][b * 16 + g * 4] = o[b];
  }
  __syncthreads();
  auto joined = [&](int row, int dim, float& rr, float& ll) -> f32x4_t {
    rr = part_r[0][row];
#pragma unroll
    for (int n = 1; n < kWaves; ++n) rr = fmaxf(rr, part_r[n][row]);
    f32x4_t sum = {0, 0, 0, 0};
    ll = 0.0f;
#pragma unroll
    for (int n = 0; n < kWaves; ++n) {
      const float f = exp2_hw(reach_of(part_r[n][row], rr, a.scale));
      ll += f * part_l[n][row];
      sum += f * *(const f32x4_t*)&part[n][row][dim];
    }
    return sum;
  };
  auto put = [&](int row, int dim, f32x4_t v, float ll) {
    const int t = row / group;
    T* out = (T*)a.out + (int64_t)(w.row + t) * a.ldo + (int64_t)(h * group + row - t * group) * d + dim;
    const float inv = 1.0f / ll;
    *(uint64_t*)out = (uint64_t)pack2<T>(v[0] * inv, v[1] * inv) | ((uint64_t)pack2<T>(v[2] * inv, v[3] * inv) << 32);
  };
  const int quads = rows * (d / 4);
  if (splits == 1) {
    for (int e = threadIdx.x; e < quads; e += kThreads) {
      const int row = e / (d / 4), dim = (e - row * (d / 4)) * 4;
      float rr, ll;
      const f32x4_t v = joined(row, dim, rr, ll);
      put(row, dim, v, ll);
    }
    return;
  }
  // a part: [rows][d] sums, then [rows] pairs of reference and weight sum
  float* parts = p.parts + ((int64_t)w.slot * kv_heads + h) * p.slot_floats;
  const int64_t pitch = (int64_t)kv_heads * p.slot_floats;
  float* mine = parts + w.split * pitch;
  for (int e = threadIdx.x; e < quads; e += kThreads) {
    const int row = e / (d / 4), dim = (e - row * (d / 4)) * 4;
    float rr, ll;
    const f32x4_t v = joined(row, dim, rr, ll);
    store_pair(mine + row * d + dim, v[0], v[1]);
    store_pair(mine + row * d + dim + 2, v[2], v[3]);
    if (dim == 0) store_pair(mine + rows * d + 2 * row, rr, ll);
  }
  wait_vmem();
  __syncthreads();
  unsigned* counter = p.counters + (int64_t)w.slot * kv_heads + h;
  if (threadIdx.x == 0) flag = __hip_atomic_fetch_add(counter, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  __syncthreads();
  if (flag != (unsigned)(splits - 1)) return;
  if (threadIdx.x == 0) reset_counter(counter);
  // Threads beyond one a quad take further parts: team `team` of `teams` those at its place of every `teams`.
  const int teams = max(1, kThreads / quads);
  f32x4_t* sums = (f32x4_t*)&part[0][0][0];
  f32x2_t* heads = (f32x2_t*)(sums + kThreads);
  for (int e0 = threadIdx.x; e0 < max(quads, kThreads); e0 += kThreads) {
    const int team = e0 / quads, e = e0 - team * quads;
    const int row = e / (d / 4), dim = (e - row * (d / 4)) * 4;
    float rr = kLowest, ll = 0.0f;
    f32x4_t sum = {0, 0, 0, 0};
    constexpr int AHEAD = 8;  // parts whose loads are out together
    for (int s0 = team; s0 < splits && team < teams; s0 += AHEAD * teams) {
      f32x2_t rl[AHEAD], v0[AHEAD], v1[AHEAD];
#pragma unroll
      for (int n = 0; n < AHEAD; ++n) {
        const float* src = parts + min(s0 + n * teams, splits - 1) * pitch;
        rl[n] = load_pair(src + rows * d + 2 * row);
        v0[n] = load_pair(src + row * d + dim);
        v1[n] = load_pair(src + row * d + dim + 2);
      }
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int n = 0; n < AHEAD; ++n) {
        if (s0 + n * teams >= splits) break;
        const float now = fmaxf(rr, rl[n][0]), keep = exp2_hw(reach_of(rr, now, a.scale)), f = exp2_hw(reach_of(rl[n][0], now, a.scale));
        rr = now;
        ll = ll * keep + f * rl[n][1];
        sum = sum * keep + f * f32x4_t{v0[n][0], v0[n][1], v1[n][0], v1[n][1]};
      }
    }
    if (teams > 1) {
      sums[threadIdx.x] = sum;
      heads[threadIdx.x] = f32x2_t{rr, ll};
      __syncthreads();
      if (team) continue;
      for (int n = 1; n < teams; ++n) {
        const f32x2_t rl = heads[n * quads + e];
        const float now = fmaxf(rr, rl[0]), keep = exp2_hw(reach_of(rr, now, a.scale)), f = exp2_hw(reach_of(rl[0], now, a.scale));
        rr = now;
        ll = ll * keep + f * rl[1];
        sum = sum * keep + f * sums[n * quads + e];
      }
    }
    if (team == 0) put(row, dim, sum, ll);
  }
}

}  // namespace

}  // namespace qtts

int qtts_launch_paged_small(const qtts::PagedLaunch& p, int dtype, hipStream_t st) {
  using namespace qtts;
  const dim3 grid((uint32_t)((int64_t)p.items * p.a.cache.kv_heads + p.fill));
  auto go = [&](auto type) {
    typedef decltype(type) T;
    const int d = p.a.cache.d;
    if (d == 64) launch(paged_small_kernel<T, 64, true>, grid, dim3(kThreads), 0u, st, p);
    else if (d == 128) launch(paged_small_kernel<T, 128, true>, grid, dim3(kThreads), 0u, st, p);
    else if (d == 256) launch(paged_small_kernel<T, 256, true>, grid, dim3(kThreads), 0u, st, p);
    else if (d < 64) launch(paged_small_kernel<T, 64, false>, grid, dim3(kThreads), 0u, st, p);
    else if (d < 128) launch(paged_small_kernel<T, 128, false>, grid, dim3(kThreads), 0u, st, p);
    else launch(paged_small_kernel<T, 256, false>, grid, dim3(kThreads), 0u, st, p);
  };
  if (dtype == QTTS_BF16) go(bf16_t{});
  else go(f16_t{});
  return qtts_check_launch("paged_attention");
}
