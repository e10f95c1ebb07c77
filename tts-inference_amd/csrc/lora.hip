// Low-rank adapters of many requests beside one shared linear.  Row r of the activations carries its
// adapter's slot s = index[r] (outside [0, slots): none); with P output partitions of rank R each,
//   t[r, p R + i] = sum_c x[r, c] A[s, p R + i, c]                              (first product, "down")
//   out[r, j] = T(base[r, j] + scaling[s] sum_{i < ranks[s]} t[r, p(j) R + i] B[s, j, i])   (second, "up")
// with fp32 sums and one rounding, to the output's type.  Entries past a slot's rank are never used.
//
// Both products run on 16x16x32 MFMAs over groups of up to 16 rows that share a slot: A's rows and x's rows
// lie along K, B's rows along the rank, so an MFMA operand is 16 bytes of a row (a lane holds row lane % 16,
// elements 8 (lane / 16) ... + 7).  Loaded that way each lane is on a line of its own, and a line is touched
// at half or a quarter of its width; so x and A go to LDS in whole 128-byte lines (each wave its own part of K,
// a ring of stages without a barrier), and the result meets base in LDS, whose rows are read and written in
// 128-byte pieces.  t leaves the first product in fp32; the second multiplies it as two 16-bit halves,
// hi = T(t) and lo = T(t - hi), which keeps 16 bits of it (bf16; 22 in fp16, where the row is first scaled by
// the power of two that brings its largest entry to [1/2, 1)).
//
// Where the groups come from: up to 64 rows, each workgroup finds the rows of its slot by one load of the
// window's indices and a ballot; past them from a plan (rows sorted by slot, made once a step).
//
//  * lora_one_kernel: both products in one launch, for few adapters of small rank (lora_rule.h);
//  * lora_down_kernel, lora_up_kernel: one launch each, t through the workspace.
#include <algorithm>

#include "common.h"
#include "lora.h"
#include "lora_rule.h"
#include "pipe.h"

using namespace qtts;

namespace qtts {

static_assert(kLoraMaxParts == QTTS_LORA_MAX_PARTS && kLoraMaxRank == QTTS_LORA_MAX_RANK, "limits of the header");

template <typename XT> using vec8 = typename mfma16<XT>::vec;

// Eight elements of a row from `at`, zeros from `end` on.  VEC: the row starts on 16 bytes, at and end are multiples of 8.
template <bool VEC, typename XT> __device__ __forceinline__ i32x4_t load8(const XT* row, int at, int end) {
  i32x4_t v = {0, 0, 0, 0};
  if constexpr (VEC) {
    if (at < end) v = *(const i32x4_t*)(row + at);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t lo = at + 2 * i < end ? row[at + 2 * i].bits : 0, hi = at + 2 * i + 1 < end ? row[at + 2 * i + 1].bits : 0;
      v[i] = (int)(lo | (hi << 16));
    }
  }
  return v;
}

// ---- groups of rows ------------------------------------------------------------------------

struct Group {
  int slot;     // -1: no adapter
  int count;    // rows, at most 16
  int64_t row;  // the row of lane % 16 (of the first one past count)
};

// The group that row `at` leads among its window of 64 rows: rows of its slot, in steps of 16; count 0 for a row that
// another one leads.  A row without an adapter is a group by itself.
__device__ __forceinline__ Group group_by_ballot(const LoraArgs& g, int64_t at) {
  const int lane = threadIdx.x & 63, here = (int)(at & 63);
  const int64_t first = at - here;
  int s = first + lane < g.m ? g.index[first + lane] : -1;
  if (s < 0 || s >= g.slots) s = -1;
  const int slot = __builtin_amdgcn_readlane(s, here);
  if (slot < 0) return {-1, 1, at};
  const uint64_t same = __ballot(s == slot), below = (1ull << lane) - 1;
  const int before = __popcll(same & ((1ull << here) - 1)), total = __popcll(same);
  if (before % 16) return {slot, 0, at};
  // lane i of the window to lane `rank of i among the slot's rows` (the others past them): one permutation
  const int to = s == slot ? __popcll(same & below) : total + __popcll(~same & below);
  const int order = __builtin_amdgcn_ds_permute(4 * to, lane);
  const int count = min(16, total - before), j = lane & 15;
  return {slot, count, first + __builtin_amdgcn_ds_bpermute(4 * (before + (j < count ? j : 0)), order)};
}

// Sub-group `sub` (16 rows) of tile `tile` < plan_max_tiles; count 0 past its end, past the plan's tiles and where the
// plan was made for another batch or slot count.
__device__ __forceinline__ Group group_by_plan(const LoraArgs& g, int64_t tile, int sub) {
  const i32x4_t head = *(const i32x4_t*)g.plan, e = *(const i32x4_t*)(g.plan + 4 + 4 * tile);
  const int count = min(16, e[2] - 16 * sub), j = threadIdx.x & 15;
  if (tile >= head[0] || head[1] != g.m || head[2] != g.slots || count <= 0) return {-1, 0, 0};
  const int64_t at = plan_order_at(g.m, g.slots) + e[1] + 16 * sub + (j < count ? j : 0);
  return {e[0], count, g.plan[at]};
}

__device__ __forceinline__ int live_rank(const LoraArgs& g, int slot) {
  return g.ranks ? min(max(g.ranks[slot], 0), g.rank) : g.rank;
}

// ---- first product ---------------------------------------------------------------------------

// Stages of a wave's ring: 64 of K of the group's rows and of N 16-row tiles of A, each tile two direct loads of 1 KiB
// (eight rows of 128 bytes, pieces swizzled as pipe.h's stages).
template <int N> constexpr int kDownStages = N == 1 ? 4 : N == 2 ? 3 : 2;
template <int N> constexpr int kDownBytes = kDownStages<N> * (N + 1) * 2048;  // of a wave

// Rows [row0, row0 + 16 N) of a slot's A by the group's rows, over K from 32 s0 to 32 s1 (s0 even):
// acc[i] holds, in lane l, rows 16 i + 4 (l / 16) ... + 3 of A for the group's row l % 16.  Rows past the slot's rank, or past
// `rows`, give values that nothing reads.  lds: kDownBytes<N> of this wave alone.
template <typename XT, int N, bool VEC>
__device__ __forceinline__ void down_steps(const LoraArgs& g, const Group& gr, const XT* a, int row0, int rows, int live, int s0,
                                           int s1, uint8_t* lds, f32x4_t* acc) {
  const int lane = threadIdx.x & 63, j = lane & 15, q = lane >> 4;
  if constexpr (VEC) {
    constexpr int S = kDownStages<N>, L = 2 * (N + 1);  // direct loads a stage
    const XT* from[L];  // each direct load's row and piece, at K = 0
#pragma unroll
    for (int i = 0; i < L; ++i) {
      const int r = (i & 1) * 8 + (lane >> 3), piece = 8 * swizzle8(r, lane & 7);
      if (i < 2) {
        const int row = __builtin_amdgcn_ds_bpermute(4 * r, (int)gr.row);
        from[i] = (const XT*)g.x + (int64_t)row * g.ldx + piece;
      } else {  // hidden rows read the first one: in cache
        const int ar = row0 + 16 * ((i - 2) >> 1) + r;
        from[i] = a + (int64_t)(ar < rows && ar % g.rank < live ? ar : 0) * g.k + piece;
      }
    }
    const int c1 = (s1 + 1) >> 1, tail = g.k - 8;
    auto issue = [&](int c) {
      uint8_t* stage = lds + c % S * (L * 1024);
#pragma unroll
      for (int i = 0; i < L; ++i) {
        const int r = (i & 1) * 8 + (lane >> 3), p = 8 * swizzle8(r, lane & 7);
        const int past = max(64 * c + p - tail, 0);  // a piece past K: the row's last one, zeroed when it is read
        load_to_lds16(from[i] + 64 * c - past, stage + i * 1024);
      }
    };
    int c = s0 >> 1, ahead = c;
    for (; ahead < min(c + S, c1); ++ahead) issue(ahead);
    for (; c < c1; ++c) {
      wait_stages<L, S - 1>(ahead - c - 1);
      const uint8_t* stage = lds + c % S * (L * 1024);
      i32x4_t xv[2], av[2][N];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int at = j * 128 + swizzle8(j, 4 * h + q) * 16;
        xv[h] = *(const i32x4_t*)(stage + at);
#pragma unroll
        for (int i = 0; i < N; ++i) av[h][i] = *(const i32x4_t*)(stage + 2048 * (i + 1) + at);
        if (64 * c + 32 * h + 8 * q > tail) {
          xv[h] = i32x4_t{0, 0, 0, 0};
#pragma unroll
          for (int i = 0; i < N; ++i) av[h][i] = i32x4_t{0, 0, 0, 0};
        }
      }
      wait_lgkmcnt0();  // the stage is read before it is loaded again
      if (ahead < c1) issue(ahead++);
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int i = 0; i < N; ++i)
          acc[i] = mfma16<XT>::mma(__builtin_bit_cast(vec8<XT>, av[h][i]), __builtin_bit_cast(vec8<XT>, xv[h]), acc[i]);
    }
  } else {
    const XT* x = (const XT*)g.x + gr.row * g.ldx;
    const XT* ap[N];
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int r = row0 + 16 * i + j;
      ap[i] = a + (int64_t)(r < rows && r % g.rank < live ? r : 0) * g.k;
    }
    for (int s = s0; s < s1; ++s) {
      const vec8<XT> xv = __builtin_bit_cast(vec8<XT>, load8<false>(x, 32 * s + 8 * q, g.k));
#pragma unroll
      for (int i = 0; i < N; ++i)
        acc[i] = mfma16<XT>::mma(__builtin_bit_cast(vec8<XT>, load8<false>(ap[i], 32 * s + 8 * q, g.k)), xv, acc[i]);
    }
  }
}

constexpr int kDownWaves = 4;

// Grid: (blocks of A's tiles x splits of K, groups or tiles x 4).
template <typename XT, int N, bool VEC, bool PLAN>
__global__ __launch_bounds__(64 * kDownWaves) void lora_down_kernel(LoraArgs g) {
  __shared__ __align__(1024) uint8_t stages[kDownWaves][VEC ? kDownBytes<N> : 1024 * N];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int split = blockIdx.x % g.splits, row0 = blockIdx.x / g.splits * 16 * N;
  const int64_t groups = PLAN ? 4 * plan_max_tiles(g.m, g.slots) : g.m;
  const int steps = (g.k + 31) >> 5, parts = g.splits * kDownWaves, per = ((steps + parts - 1) / parts + 1) & ~1;
  const int s0 = min((split * kDownWaves + wave) * per, steps + 1 & ~1), s1 = min(s0 + per, steps);
  for (int64_t at = blockIdx.y; at < groups; at += gridDim.y) {
    const Group gr = PLAN ? group_by_plan(g, at >> 2, (int)(at & 3)) : group_by_ballot(g, at);
    if (gr.slot < 0 || !gr.count) continue;
    const int live = live_rank(g, gr.slot);
    if (!live) continue;
    f32x4_t acc[N];
#pragma unroll
    for (int i = 0; i < N; ++i) acc[i] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
    down_steps<XT, N, VEC>(g, gr, (const XT*)g.a + (int64_t)gr.slot * g.rows_a * g.k, row0, g.rows_a, live, s0, s1,
                           stages[wave], acc);
#pragma unroll
    for (int i = 0; i < N; ++i) ((f32x4_t*)stages[wave])[64 * i + lane] = acc[i];
    __syncthreads();
    if (wave < N && (lane & 15) < gr.count && row0 + 16 * wave < g.t_stride) {
      f32x4_t v = ((f32x4_t*)stages[0])[64 * wave + lane];
#pragma unroll
      for (int w = 1; w < kDownWaves; ++w) v += ((f32x4_t*)stages[w])[64 * wave + lane];
      *(f32x4_t*)(g.t + ((int64_t)split * g.m + gr.row) * g.t_stride + row0 + 16 * wave + 4 * (lane >> 4)) = v;
    }
    __syncthreads();  // read before the next group's stages
  }
}

// ---- second product --------------------------------------------------------------------------
// The rank in blocks of 32 (NB of them).  A whole block: lane group q = lane / 16 holds entries 8 q ... + 7, and two
// MFMAs multiply them by t's high and low halves.  PACK: the last block has 16 entries or fewer, so one MFMA does
// both, groups 0-1 with the high halves and 2-3 with the low ones.

template <int NB, bool PACK> struct RankLane {
  int first[NB];  // the lane's first entry of each block
  bool low;       // PACK: the lane's half in the last block
  __device__ __forceinline__ explicit RankLane(int lane) {
    const int q = lane >> 4;
#pragma unroll
    for (int b = 0; b < NB; ++b) first[b] = 32 * b + 8 * (PACK && b == NB - 1 ? q & 1 : q);
    low = q >= 2;
  }
};

// Zeroes the entries of an operand from `at` on that are past the slot's rank: they may hold anything.
__device__ __forceinline__ i32x4_t hide(i32x4_t v, int at, int live) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int n = live - at - 2 * i;
    v[i] = n >= 2 ? v[i] : n == 1 ? v[i] & 0xffff : 0;
  }
  return v;
}

// The t operands of one group's row: (hi, lo) halves of each block, and the exponent that fp16 rows are scaled by.
template <typename XT, int NB, bool PACK> struct TOperand {
  vec8<XT> hi[NB], lo[NB];
  int exp;

  // v[b][i]: entry first[b] + i of t, scaled and zero past the slot's rank.
  __device__ __forceinline__ void set(float (&v)[NB][8], bool low) {
    exp = 0;
    if constexpr (std::is_same<XT, f16_t>::value) {
      float top = 0.0f;
#pragma unroll
      for (int b = 0; b < NB; ++b)
#pragma unroll
        for (int i = 0; i < 8; ++i) top = fmaxf(top, fabsf(v[b][i]));
      top = fmaxf(top, __shfl_xor(top, 16, 64));
      top = fmaxf(top, __shfl_xor(top, 32, 64));
      exp = __builtin_amdgcn_frexp_expf(top);  // 0 for zero, infinity and NaN
#pragma unroll
      for (int b = 0; b < NB; ++b)
#pragma unroll
        for (int i = 0; i < 8; ++i) v[b][i] = __builtin_amdgcn_ldexpf(v[b][i], -exp);
    }
#pragma unroll
    for (int b = 0; b < NB; ++b) {
      i32x4_t h, l;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        h[i] = (int)pack2_f32<XT>(v[b][2 * i], v[b][2 * i + 1]);
        const float h0 = to_f32(XT{(uint16_t)h[i]}), h1 = to_f32(XT{(uint16_t)((uint32_t)h[i] >> 16)});
        // an infinite or NaN half has no remainder
        const float l0 = fabsf(h0) <= 3.4e38f ? v[b][2 * i] - h0 : 0.0f, l1 = fabsf(h1) <= 3.4e38f ? v[b][2 * i + 1] - h1 : 0.0f;
        l[i] = (int)pack2_f32<XT>(l0, l1);
      }
      if (PACK && b == NB - 1) h = low ? l : h;  // one MFMA: the lane's half
      hi[b] = __builtin_bit_cast(vec8<XT>, h);
      lo[b] = __builtin_bit_cast(vec8<XT>, l);
    }
  }
};

// NT tiles of 16 columns a wave: lane l ends with columns c0 + 16 n + 4 (l / 16) ... + 3 of the group's row l % 16.
template <typename XT, int NB, int NT, bool PACK, bool VEC> struct UpTile {
  vec8<XT> b[NT][NB];

  __device__ __forceinline__ void load(const LoraArgs& g, int slot, int c0, int end, int live, const RankLane<NB, PACK>& rl) {
    const int i = threadIdx.x & 15;
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const int c = min(c0 + 16 * n + i, end - 1);
      const XT* row = (const XT*)g.b + ((int64_t)slot * g.n + c) * g.rank;
#pragma unroll
      for (int k = 0; k < NB; ++k) b[n][k] = __builtin_bit_cast(vec8<XT>, load8<VEC>(row, rl.first[k], g.rank));
    }
    if (live != g.rank) {
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int k = 0; k < NB; ++k)
          b[n][k] = __builtin_bit_cast(vec8<XT>, hide(__builtin_bit_cast(i32x4_t, b[n][k]), rl.first[k], live));
    }
  }

  __device__ __forceinline__ void mul(const TOperand<XT, NB, PACK>& t, f32x4_t (&acc)[NT]) const {
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      acc[n] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int k = 0; k < NB; ++k) {
        acc[n] = mfma16<XT>::mma(b[n][k], t.hi[k], acc[n]);
        if (!(PACK && k == NB - 1)) acc[n] = mfma16<XT>::mma(b[n][k], t.lo[k], acc[n]);
      }
    }
  }
};

// A group's rows of base and out, 16 NT columns of a wave: 2 NT lanes a row, eight neighbouring columns a lane, NT / 2 pieces
// a lane.  base is loaded as raw bits, in flight early.
template <typename XT, int NT, bool VEC> struct Rows {
  static constexpr int kLanes = 2 * NT, kPieces = NT / 2, kPitch = 16 * NT + 4;  // floats a row in LDS
  static constexpr int kFloats = 16 * kPitch;
  int64_t row[kPieces];
  bool live[kPieces];
  int c, end;
  i32x4_t raw[kPieces];

  // Every lane of the wave: the group's rows are read from its lanes.
  __device__ __forceinline__ void load(const LoraArgs& g, const Group& gr, int c0, int part_end) {
    const int lane = threadIdx.x & 63;
    c = c0 + 8 * (lane % kLanes), end = part_end;
#pragma unroll
    for (int h = 0; h < kPieces; ++h) {
      const int r = lane / kLanes + h * (64 / kLanes);
      row[h] = __builtin_amdgcn_ds_bpermute(4 * r, (int)gr.row);
      live[h] = r < gr.count && c < end;
      if (live[h]) raw[h] = load8<VEC>((const XT*)g.base + row[h] * g.ldb, c, end);
    }
  }

  __device__ __forceinline__ void store(const LoraArgs& g, int h, i32x4_t v) const {
    XT* out = (XT*)g.out + row[h] * g.ldo + c;
    if constexpr (VEC) {
      *(i32x4_t*)out = v;
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (c + i < end) out[i] = XT{(uint16_t)((uint32_t)v[i >> 1] >> (16 * (i & 1)))};
    }
  }

  __device__ __forceinline__ void copy(const LoraArgs& g) const {
#pragma unroll
    for (int h = 0; h < kPieces; ++h)
      if (live[h]) store(g, h, raw[h]);
  }

  // out = base + acc 2^exp, rounded once.  lds: kFloats of this wave alone.
  __device__ __forceinline__ void add(const LoraArgs& g, const f32x4_t (&acc)[NT], int exp, float* lds) const {
    const int lane = threadIdx.x & 63;
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      f32x4_t v = acc[n];
      if constexpr (std::is_same<XT, f16_t>::value)
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = __builtin_amdgcn_ldexpf(v[i], exp);
      *(f32x4_t*)(lds + (lane & 15) * kPitch + 16 * n + 4 * (lane >> 4)) = v;
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int h = 0; h < kPieces; ++h) {
      const float* from = lds + (lane / kLanes + h * (64 / kLanes)) * kPitch + 8 * (lane % kLanes);
      const f32x4_t d0 = *(const f32x4_t*)from, d1 = *(const f32x4_t*)(from + 4);
      if (!live[h]) continue;
      i32x4_t v;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t w = (uint32_t)raw[h][i];
        const float lo = i < 2 ? d0[2 * i] : d1[2 * i - 4], hi = i < 2 ? d0[2 * i + 1] : d1[2 * i - 3];
        v[i] = (int)pack2_f32<XT>(to_f32(XT{(uint16_t)w}) + lo, to_f32(XT{(uint16_t)(w >> 16)}) + hi);
      }
      store(g, h, v);
    }
  }
};

// The partition and first column of a workgroup's block of `cols` columns.
struct Block { int part, c0, end; };
__device__ __forceinline__ Block block_of(const LoraArgs& g, int chunk, int cols) {
  int p = 0;
  while (chunk >= g.parts.chunk_end[p]) ++p;  // chunk < chunk_end[count - 1]: the grid
  const int first = p ? g.parts.end[p - 1] : 0, before = p ? g.parts.chunk_end[p - 1] : 0;
  return {p, first + (chunk - before) * cols, g.parts.end[p]};
}

constexpr int kUpWaves = 4, kUpTiles = kLoraUpCols / (16 * kUpWaves), kUpGroups = 2;

// Grid: (column blocks, groups, or halves of the plan's tiles: two groups of one slot, which share the B operands).
template <typename XT, int NB, bool PACK, bool VEC, bool PLAN>
__global__ __launch_bounds__(64 * kUpWaves) void lora_up_kernel(LoraArgs g) {
  constexpr int G = PLAN ? kUpGroups : 1, NT = kUpTiles, PER = kPlanTile / 16 / G;
  typedef Rows<XT, NT, VEC> R;
  __shared__ __align__(16) float lds[kUpWaves][R::kFloats];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const Block blk = block_of(g, blockIdx.x, kLoraUpCols);
  const int c0 = blk.c0 + 16 * NT * wave, tok = lane & 15;
  if (c0 >= blk.end) return;
  const RankLane<NB, PACK> rl(lane);
  const int64_t groups = PLAN ? PER * plan_max_tiles(g.m, g.slots) : g.m;
  for (int64_t at = blockIdx.y; at < groups; at += gridDim.y) {
    Group gr[G];
#pragma unroll
    for (int i = 0; i < G; ++i)
      gr[i] = PLAN ? group_by_plan(g, at / PER, (int)(at % PER) * G + i) : group_by_ballot(g, at);
    if (!gr[0].count) continue;
    const int slot = gr[0].slot, live = slot < 0 ? 0 : live_rank(g, slot);
    if (!live && g.base == g.out) continue;
    R rows[G];
#pragma unroll
    for (int i = 0; i < G; ++i) rows[i].load(g, gr[i], c0, blk.end);
    if (!live) {
#pragma unroll
      for (int i = 0; i < G; ++i) rows[i].copy(g);
      continue;
    }
    UpTile<XT, NB, NT, PACK, VEC> up;
    up.load(g, slot, c0, blk.end, live, rl);
    const float scaling = g.scaling[slot];
#pragma unroll
    for (int i = 0; i < G; ++i) {
      if (!gr[i].count) break;
      float v[NB][8];
#pragma unroll
      for (int b = 0; b < NB; ++b)
#pragma unroll
        for (int e = 0; e < 8; ++e) v[b][e] = 0.0f;
      const float* t = g.t + gr[i].row * g.t_stride + blk.part * g.rank;
      for (int s = 0; s < g.splits; ++s, t += g.m * g.t_stride) {
#pragma unroll
        for (int b = 0; b < NB; ++b) {
          if constexpr (VEC) {
            if (rl.first[b] < live && tok < gr[i].count) {
              const f32x4_t v0 = *(const f32x4_t*)(t + rl.first[b]), v1 = *(const f32x4_t*)(t + rl.first[b] + 4);
#pragma unroll
              for (int e = 0; e < 4; ++e) v[b][e] += v0[e], v[b][4 + e] += v1[e];
            }
          } else {
#pragma unroll
            for (int e = 0; e < 8; ++e)
              if (rl.first[b] + e < live) v[b][e] += t[rl.first[b] + e];
          }
        }
      }
#pragma unroll
      for (int b = 0; b < NB; ++b)
#pragma unroll
        for (int e = 0; e < 8; ++e) v[b][e] = rl.first[b] + e < live ? v[b][e] * scaling : 0.0f;
      TOperand<XT, NB, PACK> to;
      to.set(v, rl.low);
      f32x4_t acc[NT];
      up.mul(to, acc);
      rows[i].add(g, acc, to.exp, lds[wave]);
    }
  }
}

// ---- both in one launch ----------------------------------------------------------------------

constexpr int kOneWaves = 8, kOneTiles = kLoraFusedCols / (16 * kOneWaves);

// Grid: (column blocks, rows).  The workgroup's waves share K of the first product, for its partition's rows of A alone, and
// meet in LDS; then each multiplies its own columns.
template <typename XT, int NB, bool PACK, bool VEC>
__global__ __launch_bounds__(64 * kOneWaves) void lora_one_kernel(LoraArgs g) {
  constexpr int NT = kOneTiles, N = 2 * NB - (PACK ? 1 : 0);  // 16-row tiles of A
  typedef Rows<XT, NT, VEC> R;
  constexpr int kBytes = std::max({VEC ? kDownBytes<N> : 0, 1024 * N, 4 * R::kFloats});
  __shared__ __align__(1024) uint8_t stages[kOneWaves][(kBytes + 1023) & ~1023];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const Block blk = block_of(g, blockIdx.x, kLoraFusedCols);
  const int c0 = blk.c0 + 16 * NT * wave, tok = lane & 15;
  const RankLane<NB, PACK> rl(lane);
  const int steps = (g.k + 31) >> 5, per = ((steps + kOneWaves - 1) / kOneWaves + 1) & ~1;
  const int s0 = min(wave * per, steps + 1 & ~1), s1 = min(s0 + per, steps);
  for (int64_t at = blockIdx.y; at < g.m; at += gridDim.y) {
    const Group gr = group_by_ballot(g, at);
    if (!gr.count) continue;
    const int live = gr.slot < 0 ? 0 : live_rank(g, gr.slot);
    if (!live && g.base == g.out) continue;
    R rows;
    rows.load(g, gr, c0, blk.end);
    if (!live) {
      rows.copy(g);
      continue;
    }
    UpTile<XT, NB, NT, PACK, VEC> up;
    up.load(g, gr.slot, c0, blk.end, live, rl);
    const float scaling = g.scaling[gr.slot];
    __builtin_amdgcn_sched_barrier(0);  // in flight before the ring
    f32x4_t acc1[N];
#pragma unroll
    for (int i = 0; i < N; ++i) acc1[i] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
    down_steps<XT, N, VEC>(g, gr, (const XT*)g.a + ((int64_t)gr.slot * g.rows_a + blk.part * g.rank) * g.k, 0, g.rank, live,
                           s0, s1, stages[wave], acc1);
#pragma unroll
    for (int i = 0; i < N; ++i) ((f32x4_t*)stages[wave])[64 * i + lane] = acc1[i];
    __syncthreads();
    // entries first[b] ... + 7 are rows 16 tile + 4 q' ... of two neighbouring lane groups q' of one tile
    float v[NB][8];
#pragma unroll
    for (int b = 0; b < NB; ++b) {
      const int from = 64 * (rl.first[b] >> 4) + ((rl.first[b] & 15) >> 2) * 16 + tok;
      f32x4_t lo = ((f32x4_t*)stages[0])[from], hi = ((f32x4_t*)stages[0])[from + 16];
#pragma unroll
      for (int w = 1; w < kOneWaves; ++w) lo += ((f32x4_t*)stages[w])[from], hi += ((f32x4_t*)stages[w])[from + 16];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        v[b][e] = rl.first[b] + e < live ? lo[e] * scaling : 0.0f;
        v[b][4 + e] = rl.first[b] + 4 + e < live ? hi[e] * scaling : 0.0f;
      }
    }
    TOperand<XT, NB, PACK> to;
    to.set(v, rl.low);
    f32x4_t acc[NT];
    up.mul(to, acc);
    __syncthreads();  // t is read before its place takes the result, and before the next group's stages
    rows.add(g, acc, to.exp, (float*)stages[wave]);
  }
}

// ---- the plan --------------------------------------------------------------------------------

constexpr int kPlanThreads = 1024, kPlanWaves = kPlanThreads / 64;

// f(slot, rows of this wave's window with it) for each slot among 64 rows (slots: the rows without an adapter).
template <typename F> __device__ __forceinline__ void by_slot(const int32_t* index, int64_t m, int slots, int64_t first, F&& f) {
  const int lane = threadIdx.x & 63;
  int s = slots;
  const bool in = first + lane < m;
  if (in) {
    s = index[first + lane];
    if (s < 0 || s >= slots) s = slots;
  }
  uint64_t left = __ballot(in);
  while (left) {
    const int one = __builtin_amdgcn_readlane(s, __builtin_ctzll(left));
    const uint64_t same = __ballot(in && s == one);
    f(one, same);
    left &= ~same;
  }
}

// A stable counting sort by slot in one workgroup: each wave counts a run of rows, the counts become first places, slot by
// slot and wave by wave, and the waves place their rows.
__global__ __launch_bounds__(kPlanThreads) void lora_plan_kernel(const int32_t* __restrict__ index, int64_t m, int slots,
                                                                 int32_t* __restrict__ plan) {
  extern __shared__ int32_t lds[];  // [kPlanWaves][slots + 1] counts, then places; [slots + 1] rows, first rows, first tiles
  const int n = slots + 1, tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  int32_t *rows = lds + kPlanWaves * n, *first_row = rows + n, *first_tile = first_row + n;
  for (int i = tid; i < kPlanWaves * n; i += kPlanThreads) lds[i] = 0;
  __syncthreads();
  const int64_t run = (m + 64 * kPlanWaves - 1) / (64 * kPlanWaves) * 64;
  const int64_t r0 = wave * run, r1 = r0 + run < m ? r0 + run : m;
  int32_t* mine = lds + wave * n;
  for (int64_t r = r0; r < r1; r += 64)
    by_slot(index, m, slots, r, [&](int s, uint64_t same) {
      if (lane == 0) mine[s] += __popcll(same);
    });
  __syncthreads();
  for (int s = tid; s < n; s += kPlanThreads) {
    int total = 0;
    for (int w = 0; w < kPlanWaves; ++w) total += lds[w * n + s];
    rows[s] = total;
  }
  __syncthreads();
  if (wave == 0) {  // exclusive sums over the slots
    int row = 0, tile = 0;
    for (int s0 = 0; s0 < n; s0 += 64) {
      const int c = s0 + lane < n ? rows[s0 + lane] : 0, t = (c + kPlanTile - 1) / kPlanTile;
      int cs = c, ts = t;
#pragma unroll
      for (int o = 1; o < 64; o <<= 1) {
        const int cu = __shfl_up(cs, o, 64), tu = __shfl_up(ts, o, 64);
        if (lane >= o) cs += cu, ts += tu;
      }
      if (s0 + lane < n) first_row[s0 + lane] = row + cs - c, first_tile[s0 + lane] = tile + ts - t;
      row += __shfl(cs, 63, 64);
      tile += __shfl(ts, 63, 64);
    }
    if (lane == 0) plan[0] = tile, plan[1] = (int32_t)m, plan[2] = slots;
  }
  __syncthreads();
  for (int s = tid; s < n; s += kPlanThreads) {
    const int total = rows[s], start = first_row[s], tile = first_tile[s];
    for (int i = 0; i * kPlanTile < total; ++i)
      *(i32x4_t*)(plan + 4 + 4 * (int64_t)(tile + i)) =
          i32x4_t{s < slots ? s : -1, start + i * kPlanTile, min(kPlanTile, total - i * kPlanTile), 0};
    int place = start;
    for (int w = 0; w < kPlanWaves; ++w) {
      const int c = lds[w * n + s];
      lds[w * n + s] = place;
      place += c;
    }
  }
  __syncthreads();
  int32_t* order = plan + plan_order_at(m, slots);
  for (int64_t r = r0; r < r1; r += 64)
    by_slot(index, m, slots, r, [&](int s, uint64_t same) {
      int place = 0;
      if (lane == 0) place = mine[s], mine[s] = place + __popcll(same);  // lane 0 alone reads and writes the wave's places
      place = __builtin_amdgcn_readfirstlane(place);
      if (same >> lane & 1) order[place + __popcll(same & ((1ull << lane) - 1))] = (int32_t)(r + lane);
    });
}

}  // namespace qtts

namespace {

constexpr unsigned kMaxGridY = 65535;

unsigned grid_y(int64_t n) { return (unsigned)std::min<int64_t>(n, kMaxGridY); }

// f(NB, PACK) of a rank, as constants.
template <typename F> void by_rank(int rank, F&& f) {
  using std::integral_constant;
  if (rank <= 16) f(integral_constant<int, 1>{}, std::true_type{});
  else if (rank <= 32) f(integral_constant<int, 1>{}, std::false_type{});
  else if (rank <= 48) f(integral_constant<int, 2>{}, std::true_type{});
  else if (rank <= 64) f(integral_constant<int, 2>{}, std::false_type{});
  else if (rank <= 96) f(integral_constant<int, 3>{}, std::false_type{});
  else f(integral_constant<int, 4>{}, std::false_type{});
}

template <typename F> void by_bool(bool v, F&& f) {
  if (v) f(std::true_type{});
  else f(std::false_type{});
}

// Column blocks of `cols` columns, none across a partition's end.
int cut_columns(LoraParts& parts, int cols) {
  int chunks = 0;
  for (int p = 0; p < parts.count; ++p) {
    chunks += (parts.end[p] - (p ? parts.end[p - 1] : 0) + cols - 1) / cols;
    parts.chunk_end[p] = chunks;
  }
  return chunks;
}

bool aligned(const void* p, int64_t ld) { return (uintptr_t)p % 16 == 0 && ld % 8 == 0; }

template <typename XT> void launch_lora(LoraArgs& g, hipStream_t st) {
  // The operands of each product as 16-byte vectors: its rows start on 16 bytes and its widths are multiples of 8.
  const bool vec_k = g.k % 8 == 0 && aligned(g.x, g.ldx) && aligned(g.a, 0);
  bool vec_n = g.rank % 8 == 0 && aligned(g.b, 0) && aligned(g.base, g.ldb) && aligned(g.out, g.ldo);
  for (int p = 0; p < g.parts.count; ++p) vec_n = vec_n && g.parts.end[p] % 8 == 0;
  const int chunks = cut_columns(g.parts, kLoraFusedCols);
  if (lora_one_launch(g.plan, g.m, g.k, g.rank, g.slots, chunks)) {
    by_rank(g.rank, [&](auto nb, auto pack) {
      if constexpr (32 * nb.value <= kLoraOneRank)
        by_bool(vec_k && vec_n, [&](auto v) {
          qtts::launch(&lora_one_kernel<XT, nb.value, pack.value, v.value>, dim3(chunks, grid_y(g.m)), dim3(64 * kOneWaves), 0,
                       st, g);
        });
    });
    return;
  }
  const int64_t tiles = g.plan ? plan_max_tiles(g.m, g.slots) : g.m;
  const int n = std::min((g.rows_a + 15) / 16, kLoraAtiles), blocks = (g.rows_a + 16 * n - 1) / (16 * n);
  by_bool(g.plan, [&](auto plan) {
    by_bool(vec_k, [&](auto v) {
      const dim3 grid(blocks * g.splits, grid_y(plan.value ? 4 * tiles : tiles)), block(64 * kDownWaves);
      if (n == 1) qtts::launch(&lora_down_kernel<XT, 1, v.value, plan.value>, grid, block, 0, st, g);
      else if (n == 2) qtts::launch(&lora_down_kernel<XT, 2, v.value, plan.value>, grid, block, 0, st, g);
      else if (n == 3) qtts::launch(&lora_down_kernel<XT, 3, v.value, plan.value>, grid, block, 0, st, g);
      else qtts::launch(&lora_down_kernel<XT, 4, v.value, plan.value>, grid, block, 0, st, g);
    });
    const int up_chunks = cut_columns(g.parts, kLoraUpCols);
    by_rank(g.rank, [&](auto nb, auto pack) {
      by_bool(vec_n, [&](auto v) {
        qtts::launch(&lora_up_kernel<XT, nb.value, pack.value, v.value, plan.value>, dim3(up_chunks, grid_y(plan.value ? kPlanTile / 16 / kUpGroups * tiles : tiles)),
                     dim3(64 * kUpWaves), 0, st, g);
      });
    });
  });
}

}  // namespace

int64_t qtts_lora_ws_bytes(int64_t m, int64_t rows_a, int64_t k) {
  return kCounterBytes + align256(lora_splits(m, rows_a, k) * m * lora_t_stride(rows_a) * 4);
}

int64_t qtts_lora_plan_words(int64_t m, int64_t slots) { return slots <= kPlanMaxSlots ? plan_words(m, slots) : 0; }

int qtts_launch_lora_plan(const int32_t* index, int64_t m, int64_t slots, int32_t* plan, hipStream_t st) {
  const uint32_t shmem = (uint32_t)((kPlanWaves + 3) * (slots + 1) * 4);
  qtts::launch(&lora_plan_kernel, dim3(1), dim3(kPlanThreads), shmem, st, index, m, slots, plan);
  return qtts_check_launch("lora_plan");
}

int qtts_launch_lora_add(const LoraArgs& args, int x_dtype, void* ws, hipStream_t st) {
  LoraArgs g = args;
  g.t = (float*)((char*)ws + kCounterBytes);
  g.rows_a = g.parts.count * g.rank;
  g.t_stride = (int)lora_t_stride(g.rows_a);
  g.splits = lora_splits(g.m, g.rows_a, g.k);
  if (x_dtype == QTTS_BF16) launch_lora<bf16_t>(g, st);
  else launch_lora<f16_t>(g, st);
  return qtts_check_launch("lora_add");
}
