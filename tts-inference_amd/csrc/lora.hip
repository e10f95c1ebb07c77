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
// 128-byte pieces.
//
// The second product multiplies t, scaled, as 16-bit parts, each the rounding of what those before it leave: in bf16
// three, which hold all 24 bits of fp32 (with two, 16 bits, an adapter whose terms cancel lost the rest; the third costs a
// layer of 27 rows 0.7%, of 2048 2.8%, ranks past 16 and many rows 4-5%); in fp16 two, 22 bits of entries down to
// 2^-17 of the largest of each 32, which are first scaled by a power of two.
// The first product's kernel writes them so: the second, whose time is the output's rows, only loads them.
//
// Where the groups come from: up to 64 rows, each workgroup finds the rows of its slot by one load of the
// window's indices and a ballot; past them from a plan (rows sorted by slot, made once a step).
//
//  * lora_one_kernel: both products in one launch, for few adapters of small rank (lora_rule.h);
//  * lora_down_kernel, lora_up_kernel: one launch each, t through the workspace.
//
// What bounds them, bf16 (a large copy runs at 5.1 TB/s here; each figure a kernel's own time, its inputs from memory, and in
// brackets with the same inputs in every call, which the Infinity Cache then holds):
//  * one launch: latency, three round trips to memory (the index; x, A, B and base; the result).  Rank 16, one row through 2048 x
//    2048 in 5.7 us (5.5), 27 rows of 9 adapters through 2048 -> 12288 in 8.3 (7.9): 4.7 MB of A and B;
//  * the first product: its groups' loads of x and A, each group's anew.  64 rows of 32 rank-64 adapters, two partitions of 2048
//    (17 MB of A), in 8.2 us (7.3); 2048 rows of 8 rank-16 adapters, K = 2048, in 7.3 (8 MB of x, 19 MB through the L2s), K = 6144 in
//    13.0 (25 and 53), by 137 workgroups, which is why K's parts and A's tiles get workgroups of their own while groups are few.
//    Past rank 32 and a thousand rows A's re-reads: 4096 rows through qkv, rank 64, 8 adapters 34 us (276 MB through the L2s, 40%
//    of them missed), 64 adapters 50 (297 MB, 94%);
//  * the second product: base and the result, or B where rows are few.  2048 rows through 2048 -> 12288, rank 16, in 25.8 us (19.7):
//    101 MB, 3.9 TB/s; 64 rows of 32 rank-64 adapters (50 MB of B) in 14.6 (11.6).
#include <algorithm>

#include "common.h"
#include "lora.h"
#include "lora_rule.h"
#include "pipe.h"

using namespace qtts;

namespace qtts {

typedef __attribute__((ext_vector_type(2))) int i32x2_t;

static_assert(kLoraMaxParts == QTTS_LORA_MAX_PARTS && kLoraMaxRank == QTTS_LORA_MAX_RANK, "limits of the header");

template <typename XT> using vec8 = typename mfma16<XT>::vec;

// Eight elements of a row from `at`, one by one; zeros from `end` on (the last one is read again there).
template <typename XT> __device__ __forceinline__ i32x4_t load8(const XT* row, int at, int end) {
  i32x4_t v;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int e0 = at + 2 * i, e1 = e0 + 1;
    const uint32_t lo = row[min(e0, end - 1)].bits, hi = row[min(e1, end - 1)].bits;
    v[i] = (int)((e0 < end ? lo : 0) | (e1 < end ? hi << 16 : 0));
  }
  return v;
}

// ---- groups of rows ------------------------------------------------------------------------

struct Group {
  int slot;     // -1: no adapter
  int count;    // rows, at most 16
  int64_t row;  // the row of lane % 16 (of the first one past count)
};

// The lanes of `in` whose slot (0 to slots) is this lane's, bit by bit of the slot (a loop over the slots among 64 rows waits 90 ns
// or more for each).
__device__ __forceinline__ uint64_t same_slot(int slot, int slots, bool in) {
  uint64_t same = __ballot(in);
  for (int bit = 1; bit <= slots; bit <<= 1) {
    const uint64_t set = __ballot((slot & bit) != 0);
    same &= slot & bit ? set : ~set;
  }
  return same;
}

// Group `at` without a plan, count 0 for none; every 16th row of a slot among 64 rows leads one.  With a place for each row
// (g.groups == g.m) it is the one that row `at` leads; with fewer, of up to 64 rows, the at-th in the order of their first rows.
__device__ __forceinline__ Group group_by_ballot(const LoraArgs& g, int64_t at) {
  const int lane = threadIdx.x & 63;
  const int64_t window = at & ~(int64_t)63;
  const uint64_t below = (1ull << lane) - 1;
  const bool in = window + lane < g.m;
  int s = in ? g.index[window + lane] : -1;
  if (s < 0 || s >= g.slots) s = g.slots;
  int leader = (int)(at & 63);
  if (g.groups < g.m) {
    const uint64_t leaders = __ballot(in && __popcll(same_slot(s, g.slots, in) & below) % 16 == 0);
    const uint64_t found = __ballot((leaders >> lane & 1) && __popcll(leaders & below) == leader);
    if (!found) return {-1, 0, 0};
    leader = __builtin_ctzll(found);
  }
  const int slot = __builtin_amdgcn_readlane(s, leader);
  const uint64_t same = __ballot(in && s == slot);
  const int total = __popcll(same), before = __popcll(same & ((1ull << leader) - 1));
  if (before % 16) return {-1, 0, 0};
  // lane i of the window to lane `rank of i among the slot's rows` (the others past them): one permutation
  const int to = same >> lane & 1 ? __popcll(same & below) : total + __popcll(~same & below);
  const int order = __builtin_amdgcn_ds_permute(4 * to, lane);
  const int count = min(16, total - before), j = lane & 15;
  return {slot < g.slots ? slot : -1, count, window + __builtin_amdgcn_ds_bpermute(4 * (before + (j < count ? j : 0)), order)};
}

// Group `at` < plan_max_groups of the plan; count 0 past the plan's groups, -1 where the plan was made for another batch or
// slot count.  The three loads do not wait for one another.
__device__ __forceinline__ Group group_by_plan(const LoraArgs& g, int64_t at) {
  const int j = threadIdx.x & 15;
  const i32x4_t head = *(const i32x4_t*)g.plan;
  const i32x2_t e = *(const i32x2_t*)(g.plan + 4 + 2 * at);
  const int32_t* order = g.plan + plan_order_at(g.m, g.slots) + kPlanGroup * at;
  const int row = order[j], lead = order[0];
  if (head[1] != g.m || head[2] != g.slots) return {-1, -1, 0};
  if (at >= head[0]) return {-1, 0, 0};
  return {e[0], e[1], j < e[1] ? row : lead};
}

// The slots' ranks: the first 64 by lane, loaded beside what names the slot.
struct Ranks {
  int mine;
  __device__ __forceinline__ explicit Ranks(const LoraArgs& g) {
    const int lane = threadIdx.x & 63;
    mine = g.ranks && lane < g.slots ? g.ranks[lane] : g.rank;
  }
  __device__ __forceinline__ int of(const LoraArgs& g, int slot) const {
    if (slot < 0) return 0;
    const int r = slot < 64 ? __builtin_amdgcn_readlane(mine, slot) : g.ranks ? g.ranks[slot] : g.rank;
    return min(max(r, 0), g.rank);
  }
};

// ---- first product ---------------------------------------------------------------------------

// Stages of a wave's ring: 64 of K of the group's rows and of N 16-row tiles of A, each tile two direct loads of 1 KiB
// (eight rows of 128 bytes, pieces swizzled as pipe.h's stages).
template <int N> constexpr int kDownStages = N == 1 ? 4 : N == 2 ? 3 : 2;
template <int N, int S> constexpr int kDownBytes = S * (N + 1) * 2048;  // of a wave

// N 16-row tiles of a slot's A, row(i, j) the j-th row of tile i (rows past the slot's rank give values that nothing
// reads, and are taken from its first row, which is in cache), by the group's rows, over K from 32 s0 to 32 s1
// (s0 even): acc[i] holds, in lane l, rows 4 (l / 16) ... + 3 of tile i for the group's row l % 16.  lds: kDownBytes<N, S> of
// this wave alone.
template <typename XT, int N, int S, bool VEC, typename F>
__device__ __forceinline__ void down_steps(const LoraArgs& g, const Group& gr, const XT* a, F&& row, int s0, int s1,
                                           uint8_t* lds, f32x4_t* acc) {
  const int lane = threadIdx.x & 63, j = lane & 15, q = lane >> 4;
  if constexpr (VEC) {
    constexpr int L = 2 * (N + 1);  // direct loads a stage
    const XT* from[L];              // each direct load's row and piece, at the next stage's K
    const int c0 = s0 >> 1, c1 = (s1 + 1) >> 1, whole = min(c1, g.k >> 6);
#pragma unroll
    for (int i = 0; i < L; ++i) {
      const int r = (i & 1) * 8 + (lane >> 3), at = 64 * c0 + 8 * swizzle8(r, lane & 7);
      if (i < 2) from[i] = (const XT*)g.x + (int64_t)__builtin_amdgcn_ds_bpermute(4 * r, (int)gr.row) * g.ldx + at;
      else from[i] = a + (int64_t)row((i - 2) >> 1, r) * g.k + at;
    }
    int into = 0, out = 0, ahead = c0;  // stages of the ring
    auto issue = [&]() {
#pragma unroll
      for (int i = 0; i < L; ++i) {
        load_to_lds16(from[i], lds + (into * L + i) * 1024);
        from[i] += 64;
      }
      into = into + 1 == S ? 0 : into + 1;
      ++ahead;
    };
    i32x4_t xv[2], av[2][N];
    auto read = [&](const uint8_t* stage) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int at = j * 128 + swizzle8(j, 4 * h + q) * 16;
        xv[h] = *(const i32x4_t*)(stage + at);
#pragma unroll
        for (int i = 0; i < N; ++i) av[h][i] = *(const i32x4_t*)(stage + 2048 * (i + 1) + at);
      }
    };
    auto multiply = [&]() {
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int i = 0; i < N; ++i)
          acc[i] = mfma16<XT>::mma(__builtin_bit_cast(vec8<XT>, av[h][i]), __builtin_bit_cast(vec8<XT>, xv[h]), acc[i]);
    };
    while (ahead < min(c0 + S, whole)) issue();
    for (int c = c0; c < whole; ++c) {
      wait_stages<L, S - 1>(ahead - c - 1);
      read(lds + out * (L * 1024));
      out = out + 1 == S ? 0 : out + 1;
      wait_lgkmcnt0();  // the stage is read before it is loaded again
      if (ahead < whole) issue();
      multiply();
    }
    if (max(c0, whole) < c1) {  // the last stage of a K that is no multiple of 64: its missing pieces are zeros
      const int left = g.k - 64 * whole;  // of K, a multiple of 8
#pragma unroll
      for (int i = 0; i < L; ++i) {
        const int piece = 8 * swizzle8((i & 1) * 8 + (lane >> 3), lane & 7);
        load_to_lds16(from[i] - (piece < left ? 0 : piece), lds + i * 1024);
      }
      wait_vmcnt<0>();
      read(lds);
#pragma unroll
      for (int h = 0; h < 2; ++h)
        if (32 * h + 8 * q >= left) {
          xv[h] = i32x4_t{0, 0, 0, 0};
#pragma unroll
          for (int i = 0; i < N; ++i) av[h][i] = i32x4_t{0, 0, 0, 0};
        }
      wait_lgkmcnt0();
      multiply();
    }
  } else {
    const XT* x = (const XT*)g.x + gr.row * g.ldx;
    const XT* ap[N];
#pragma unroll
    for (int i = 0; i < N; ++i) ap[i] = a + (int64_t)row(i, j) * g.k;
    for (int s = s0; s < s1; ++s) {
      const vec8<XT> xv = __builtin_bit_cast(vec8<XT>, load8(x, 32 * s + 8 * q, g.k));
#pragma unroll
      for (int i = 0; i < N; ++i)
        acc[i] = mfma16<XT>::mma(__builtin_bit_cast(vec8<XT>, load8(ap[i], 32 * s + 8 * q, g.k)), xv, acc[i]);
    }
  }
}

// ---- t's parts -------------------------------------------------------------------------------
// The rank in blocks: up to 16 entries one block of 16 (PACK), past them NB blocks of 32.  A block of a row in the workspace: its
// parts, one after another.  A lane's operands, one an MFMA: whole blocks, entries 8 (lane / 16) ... + 7 of each part; PACK, the
// first part for lanes 0-31 and the second for lanes 32-63, then the third for lanes 0-31 alone.

template <typename XT> constexpr int kParts = std::is_same<XT, f16_t>::value ? 2 : 3;
template <bool PACK> constexpr int kBlockTiles = PACK ? 1 : 2;
template <bool PACK> constexpr int kPartBytes = PACK ? 32 : 64;
template <typename XT, bool PACK> constexpr int kBlockBytes = kParts<XT> * kPartBytes<PACK>;
template <typename XT, bool PACK> constexpr int kOperands = PACK ? (kParts<XT> + 1) / 2 : kParts<XT>;

// Operand h of a block.
template <bool PACK> __device__ __forceinline__ i32x4_t load_part(const uint8_t* block, int h) {
  const int q = (threadIdx.x & 63) >> 4;
  if (!PACK || h == 0) return *(const i32x4_t*)(block + 64 * h + 16 * q);
  const i32x4_t v = *(const i32x4_t*)(block + 64 + 16 * (q & 1));
  return q < 2 ? v : i32x4_t{0, 0, 0, 0};
}

// Four neighbouring entries of t (already zero past the slot's rank) as parts, to their place in a block.
template <typename XT, bool PACK> __device__ __forceinline__ void store_parts(f32x4_t v, uint8_t* to) {
#pragma unroll
  for (int p = 0; p < kParts<XT>; ++p) {
    uint32_t h[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      h[i] = pack2_f32<XT>(v[2 * i], v[2 * i + 1]);
      const float h0 = to_f32(XT{(uint16_t)h[i]}), h1 = to_f32(XT{(uint16_t)(h[i] >> 16)});
      // an infinite part leaves nothing
      v[2 * i] = fabsf(h0) <= 3.4e38f ? v[2 * i] - h0 : 0.0f, v[2 * i + 1] = fabsf(h1) <= 3.4e38f ? v[2 * i + 1] - h1 : 0.0f;
    }
    *(uint2*)(to + p * kPartBytes<PACK>) = make_uint2(h[0], h[1]);
  }
}

// fp16: the exponent that brings the largest of a block's entries to [2^14, 2^15) (four lanes a row), and the entries scaled by it: as
// far up as halves go, so that entries down to 2^-17 of it keep 22 bits and to 2^-28 the first part's 11.
template <typename XT, int T> __device__ __forceinline__ int scale_block(f32x4_t (&v)[T]) {
  if constexpr (!std::is_same<XT, f16_t>::value) return 0;
  float top = 0.0f;
#pragma unroll
  for (int t = 0; t < T; ++t)
#pragma unroll
    for (int i = 0; i < 4; ++i) top = fmaxf(top, fabsf(v[t][i]));
  top = fmaxf(top, __shfl_xor(top, 16, 64));
  top = fmaxf(top, __shfl_xor(top, 32, 64));
  const int exp = top < __builtin_inff() ? __builtin_amdgcn_frexp_expf(top) - 15 : 0;  // (an infinity's finite neighbours as they are)
#pragma unroll
  for (int t = 0; t < T; ++t)
#pragma unroll
    for (int i = 0; i < 4; ++i) v[t][i] = __builtin_amdgcn_ldexpf(v[t][i], -exp);
  return exp;
}

// Tiles [tile, tile + T) of the waves' sums in LDS (wave w's at sums + w * pitch bytes), added, scaled, zero past the rank;
// r0: the first tile's first entry of its partition.
template <int W, int T>
__device__ __forceinline__ void meet_waves(const uint8_t* sums, int pitch, int tile, int r0, int live, float scaling,
                                           f32x4_t (&v)[T]) {
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int t = 0; t < T; ++t) {
    v[t] = *(const f32x4_t*)(sums + (64 * (tile + t) + lane) * 16);
#pragma unroll
    for (int w = 1; w < W; ++w) v[t] += *(const f32x4_t*)(sums + w * pitch + (64 * (tile + t) + lane) * 16);
#pragma unroll
    for (int i = 0; i < 4; ++i) v[t][i] = r0 + 16 * t + 4 * (lane >> 4) + i < live ? v[t][i] * scaling : 0.0f;
  }
}

// Both products of rows `row`, row + step, ..., from the index: what a call that writes every row falls back on where its plan is
// another batch's (a captured step replayed after the routing of other rows).  Row by row and in fp32.  It is in the first product's
// kernel, whose waves a compute unit are counted by LDS: its registers, and those of groups of 16 rows in its place, cost the second's
// a wave of five, 6% of a layer of 2048 rows.  It reads the kernel's arguments anew, where the compiler does not see that they are
// those: it held them all from the kernel's start (33 scalar registers spilled, 0.4 us a launch; 0.1 so).  t: kLoraMaxRank of this
// wave alone.
template <typename XT> __device__ __forceinline__ void rows_by_index(int64_t row, int64_t step, float* t) {
  uint64_t args = (uint64_t)__builtin_amdgcn_kernarg_segment_ptr();
  asm volatile("" : "+s"(args));
  const LoraArgs& g = *(const LoraArgs*)args;
  const int lane = threadIdx.x & 63;
#pragma unroll 1
  for (; row < g.m; row += step) {
    const int slot = g.index[row];
    const bool has = slot >= 0 && slot < g.slots;
    const int live = has ? min(max(g.ranks ? g.ranks[slot] : g.rank, 0), g.rank) : 0;
    const XT *x = (const XT*)g.x + row * g.ldx, *base = (const XT*)g.base + row * g.ldb;
    XT* out = (XT*)g.out + row * g.ldo;
#pragma unroll 1
    for (int part = 0, c0 = 0; part < g.parts.count; c0 = g.parts.end[part++]) {
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");  // the last t has been read
      __builtin_amdgcn_wave_barrier();
#pragma unroll 1
      for (int i = 0; i < live; ++i) {
        const XT* a = (const XT*)g.a + (((int64_t)slot * g.parts.count + part) * g.rank + i) * g.k;
        float sum = 0.0f;
        for (int c = lane; c < g.k; c += 64) sum = __builtin_fmaf(to_f32(x[c]), to_f32(a[c]), sum);
        sum = wave_sum(sum);
        if (lane == 0) t[i] = sum * g.scaling[slot];
      }
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      __builtin_amdgcn_wave_barrier();
#pragma unroll 1
      for (int c = c0 + lane; c < g.parts.end[part]; c += 64) {
        const XT* b = (const XT*)g.b + ((int64_t)slot * g.n + c) * g.rank;  // (not read without a slot)
        float sum = 0.0f;
        for (int i = 0; i < live; ++i) sum = __builtin_fmaf(t[i], to_f32(b[i]), sum);
        out[c] = live ? from_f32<XT>(to_f32(base[c]) + sum) : base[c];
      }
    }
  }
}

constexpr int kDownWaves = 8;

// Grid: (N tiles of the partitions' A each, groups, splits of K).  Eight waves share the split's K.
template <typename XT, int N, bool PACK, bool VEC, bool PLAN>
__global__ __launch_bounds__(64 * kDownWaves) void lora_down_kernel(LoraArgs g) {
  constexpr int T = kBlockTiles<PACK>, kPitch = VEC ? kDownBytes<N, kDownStages<N>> : 1024 * N;
  static_assert(kLoraMaxRank * 4 <= kPitch, "rows_by_index");
  __shared__ __align__(1024) uint8_t stages[kDownWaves][kPitch];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int per_part = T * g.blocks, tile0 = blockIdx.x * N;  // tiles of a partition; the workgroup's first
  const Ranks ranks(g);
  const int cuts = kDownWaves * g.splits, steps = (g.k + 31) >> 5, per = ((steps + cuts - 1) / cuts + 1) & ~1;
  const int s0 = min((int)(kDownWaves * blockIdx.z + wave) * per, (steps + 1) & ~1), s1 = min(s0 + per, steps);
  for (int64_t at = blockIdx.y; at < g.groups; at += gridDim.y) {
    const Group gr = PLAN ? group_by_plan(g, at) : group_by_ballot(g, at);
    if (PLAN && gr.count < 0) {  // for every group: each workgroup is here once, the second product's not at all
      if (g.whole && blockIdx.x == 0 && blockIdx.z == 0)
        rows_by_index<XT>((int64_t)blockIdx.y * kDownWaves + wave, (int64_t)gridDim.y * kDownWaves, (float*)stages[wave]);
      return;
    }
    if (!gr.count) continue;
    const int live = ranks.of(g, gr.slot);
    if (!live) continue;
    f32x4_t acc[N];
#pragma unroll
    for (int i = 0; i < N; ++i) acc[i] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
    const float scaling = g.scaling[gr.slot];
    auto row = [&](int i, int j) {
      const int part = (tile0 + i) / per_part, r = 16 * ((tile0 + i) % per_part) + j;
      return part < g.parts.count && r < live ? part * g.rank + r : 0;
    };
    down_steps<XT, N, kDownStages<N>, VEC>(g, gr, (const XT*)g.a + (int64_t)gr.slot * g.parts.count * g.rank * g.k, row, s0,
                                           s1, stages[wave], acc);
#pragma unroll
    for (int i = 0; i < N; ++i) ((f32x4_t*)stages[wave])[64 * i + lane] = acc[i];
    __syncthreads();
    const int tile = tile0 + T * wave;  // the wave's block
    if (wave < N / T && tile < per_part * g.parts.count) {
      f32x4_t v[T];
      meet_waves<kDownWaves, T>(stages[0], kPitch, T * wave, tile % per_part * 16, live, scaling, v);
      const int exp = scale_block<XT, T>(v);
      const int64_t block = (blockIdx.z * g.m + gr.row) * (g.parts.count * g.blocks) + tile / T;
      if ((lane & 15) < gr.count) {
        uint8_t* to = g.t + block * kBlockBytes<XT, PACK> + 8 * (lane >> 4);
#pragma unroll
        for (int t = 0; t < T; ++t) store_parts<XT, PACK>(v[t], to + 32 * t);
        if (std::is_same<XT, f16_t>::value && lane < 16) g.exps[block] = exp;
      }
    }
    __syncthreads();  // read before the next group's stages
  }
}

// ---- second product --------------------------------------------------------------------------
// The t operands of one group's rows: the parts of each block of each split's sum, and fp16's exponents.  The splits of K meet
// here, as more MFMAs by the same operand of B.
template <typename XT, int NB, bool PACK, int S = 1> struct TOperand {
  static constexpr int kEach = kOperands<XT, PACK>, kBlocks = NB * S;
  i32x4_t v[kBlocks][kEach];
  int exp[kBlocks];

  // `row`: the lane's row of the workspace (of a group's first for lanes past its rows), `part` of the partition.
  __device__ __forceinline__ void load(const LoraArgs& g, int64_t row, int part) {
#pragma unroll
    for (int b = 0; b < kBlocks; ++b) {
      const int64_t block = ((b / NB * g.m + row) * g.parts.count + part) * NB + b % NB;
#pragma unroll
      for (int h = 0; h < kEach; ++h) v[b][h] = load_part<PACK>(g.t + block * kBlockBytes<XT, PACK>, h);
      if constexpr (std::is_same<XT, f16_t>::value) exp[b] = g.exps[block];
    }
  }
};

// A slot's B by columns: an operand of 16 columns from c is the lane's eight entries of each block of rows c + lane % 16.  Read as
// 16 bytes (a lane's place as bytes in the slot's B, 32 bits: the host checks; clamped to the partition's last column), aligned where
// the rank is a multiple of 8, at any address elsewhere (gate_up of 2048 rows, rank 4: 37.5 us, rank 8, aligned, 34.6; entry by entry
// rank 4 took more than twice as long; one form for both cost rank 64 up to 6%), or entry by entry where base or out forbid vectors.
// Entries past the slot's rank may hold anything, and those past the rank are no part of the row: a lane of such entries reads others
// of its row, a rank that is no multiple of 8 has its last lane read into the next row, and all of them are masked; the last slot's
// last rows have none behind them, and are read from further ahead and shifted.  (No load is in a branch: the compiler may give each
// side of one its own copy of the MFMAs after it.)
enum { kByEntry, kAligned, kAnywhere };

struct __attribute__((packed, aligned(2))) Unaligned16 { i32x4_t v; };

// v's bytes from `back` (even, below 16) on, zeros behind.
__device__ __forceinline__ i32x4_t from_byte(i32x4_t v, uint32_t back) {
  const uint64_t lo = (uint64_t)(uint32_t)v[1] << 32 | (uint32_t)v[0], hi = (uint64_t)(uint32_t)v[3] << 32 | (uint32_t)v[2];
  const uint32_t s = 8 * (back & 7);
  const uint64_t low = lo >> s | (s ? hi << (64 - s) : 0), high = hi >> s;
  const uint64_t l = back >= 8 ? high : low, h = back >= 8 ? 0 : high;
  return i32x4_t{(int)l, (int)(l >> 32), (int)h, (int)(h >> 32)};
}

template <typename XT, int NB, bool PACK, int B> struct Columns {
  const char* slot_b;
  uint32_t at, last, step;  // of column c0 + lane % 16, of the last column, from one operand to the next
  uint32_t most;            // the last place with 16 bytes of all B from it
  int rank, c, end;
  bool masks;
  int first[NB];
  i32x4_t shown[NB];

  __device__ __forceinline__ Columns(const LoraArgs& g, int slot, int c0, int part_end, int live) {
    const int q = (threadIdx.x & 63) >> 4;
    slot_b = (const char*)((const XT*)g.b + (int64_t)slot * g.n * g.rank);
    rank = g.rank, c = c0 + (int)(threadIdx.x & 15), end = part_end;
    at = (uint32_t)c * (uint32_t)rank * 2, last = (uint32_t)(end - 1) * (uint32_t)rank * 2, step = 32 * (uint32_t)rank;
    masks = live != (PACK ? 16 : 32 * NB);
    most = slot == g.slots - 1 ? (uint32_t)g.n * (uint32_t)rank * 2 - 16 : 0xffffffffu;
#pragma unroll
    for (int b = 0; b < NB; ++b) {
      const int e = 32 * b + 8 * (PACK ? q & 1 : q);
      first[b] = B != kByEntry && e >= rank ? 0 : e;
#pragma unroll
      for (int i = 0; i < 4; ++i) shown[b][i] = live - e - 2 * i >= 2 ? -1 : live - e - 2 * i == 1 ? 0xffff : 0;
    }
  }

  // The operand of the next 16 columns.
  __device__ __forceinline__ void next(vec8<XT> (&v)[NB]) {
    i32x4_t r[NB];
    if constexpr (B != kByEntry) {
      const uint32_t from = at < last ? at : last;
#pragma unroll
      for (int b = 0; b < NB; ++b) {
        const uint32_t place = from + 2 * first[b];
        if constexpr (B == kAligned) r[b] = *(const i32x4_t*)(slot_b + place);
        else r[b] = from_byte(((const Unaligned16*)(slot_b + min(place, most)))->v, place - min(place, most));
      }
      at += step;
    } else {
      const XT* row = (const XT*)slot_b + (int64_t)min(c, end - 1) * rank;
#pragma unroll
      for (int b = 0; b < NB; ++b) r[b] = load8(row, first[b], rank);
      c += 16;
    }
#pragma unroll
    for (int b = 0; b < NB; ++b) {
      if (masks) r[b] &= shown[b];
      v[b] = __builtin_bit_cast(vec8<XT>, r[b]);
    }
  }
};

template <typename XT, int NB, bool PACK, int S>
__device__ __forceinline__ f32x4_t up_mma(const vec8<XT> (&b)[NB], const TOperand<XT, NB, PACK, S>& t) {
  f32x4_t sum = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
  for (int k = 0; k < NB * S; ++k) {
    constexpr bool kExp = std::is_same<XT, f16_t>::value;  // a block at a time: each has an exponent of its own
    f32x4_t acc = kExp ? f32x4_t{0.0f, 0.0f, 0.0f, 0.0f} : sum;
#pragma unroll
    for (int h = 0; h < kOperands<XT, PACK>; ++h)
      acc = mfma16<XT>::mma(b[k % NB], __builtin_bit_cast(vec8<XT>, t.v[k][h]), acc);
    if constexpr (kExp) {
#pragma unroll
      for (int i = 0; i < 4; ++i) sum[i] += __builtin_amdgcn_ldexpf(acc[i], t.exp[k]);
    } else {
      sum = acc;
    }
  }
  return sum;
}

// A group's rows of base and out, 16 NT columns at a time: 2 NT lanes a row, eight neighbouring columns a lane, NT / 2 pieces
// a lane.  base is loaded as raw bits, in flight early.  Every lane of the wave takes part.
template <typename XT, int NT, bool VEC> struct Rows {
  static constexpr int kLanes = 2 * NT, kPieces = NT / 2, kPitch = 16 * NT + 4;  // floats a row in LDS
  static constexpr int kFloats = 16 * kPitch;
  const XT* base[kPieces];
  XT* out[kPieces];
  bool mine[kPieces];
  int c, end;
  i32x4_t raw[kPieces];

  __device__ __forceinline__ Rows(const LoraArgs& g, const Group& gr, int c0, int part_end) {
    const int lane = threadIdx.x & 63;
    c = c0 + 8 * (lane % kLanes), end = part_end;
#pragma unroll
    for (int h = 0; h < kPieces; ++h) {
      const int r = lane / kLanes + h * (64 / kLanes);
      const int64_t row = __builtin_amdgcn_ds_bpermute(4 * r, (int)gr.row);
      base[h] = (const XT*)g.base + row * g.ldb + c;
      out[h] = (XT*)g.out + row * g.ldo + c;
      mine[h] = r < gr.count;
    }
  }

  __device__ __forceinline__ void load() {
    // clamped, not in a branch: rows past the group's are its first, columns past the partition the last ones before it
#pragma unroll
    for (int h = 0; h < kPieces; ++h) {
      const int back = max(c - (end - (VEC ? 8 : 1)), 0);
      if constexpr (VEC) raw[h] = *(const i32x4_t*)(base[h] - back);
      else raw[h] = load8(base[h] - back, 0, end - c + back);
    }
  }

  __device__ __forceinline__ void store(int h, i32x4_t v) const {
    if constexpr (VEC) {
      *(i32x4_t*)out[h] = v;
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (c + i < end) out[h][i] = XT{(uint16_t)((uint32_t)v[i >> 1] >> (16 * (i & 1)))};
    }
  }

  __device__ __forceinline__ void copy() const {
#pragma unroll
    for (int h = 0; h < kPieces; ++h)
      if (mine[h] && c < end) store(h, raw[h]);
  }

  __device__ __forceinline__ void advance() {  // to the next 16 NT columns
    c += 16 * NT;
#pragma unroll
    for (int h = 0; h < kPieces; ++h) base[h] += 16 * NT, out[h] += 16 * NT;
  }

  // out = base + acc(tile), rounded once.  lds: kFloats of this wave alone.
  template <typename F> __device__ __forceinline__ void add(F&& acc, float* lds) const {
    const int lane = threadIdx.x & 63;
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");  // the last result has been read
#pragma unroll
    for (int n = 0; n < NT; ++n)
      *(f32x4_t*)(lds + (lane & 15) * kPitch + 16 * n + 4 * (lane >> 4)) = acc(n);
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
    f32x4_t d[kPieces][2];
#pragma unroll
    for (int h = 0; h < kPieces; ++h) {
      const float* from = lds + (lane / kLanes + h * (64 / kLanes)) * kPitch + 8 * (lane % kLanes);
      d[h][0] = *(const f32x4_t*)from, d[h][1] = *(const f32x4_t*)(from + 4);
    }
#pragma unroll
    for (int h = 0; h < kPieces; ++h) {
      i32x4_t v;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t w = (uint32_t)raw[h][i];
        v[i] = (int)pack2_f32<XT>(to_f32(XT{(uint16_t)w}) + d[h][i >> 1][2 * (i & 1)],
                                  to_f32(XT{(uint16_t)(w >> 16)}) + d[h][i >> 1][2 * (i & 1) + 1]);
      }
      if (mine[h] && c < end) store(h, v);
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

constexpr int kUpWaves = 4, kUpTiles = 4, kUpBlock = 16 * kUpTiles;

// Grid: (blocks of g.up_cols columns, groups).  A wave takes 64 columns at a time: with a plan, whose groups of one slot follow
// one another, all columns of a group of its own; else a part of the workgroup's group.  ONE (with a plan): those are 64 and no more,
// which without the next ones' loads takes 12 registers less (2048 rows of a layer 76.8 -> 75.2 us).
template <typename XT, int NB, bool PACK, int B, bool PLAN, int S, bool ONE>
__global__ __launch_bounds__(64 * kUpWaves) void lora_up_kernel(LoraArgs g) {
  typedef Rows<XT, kUpTiles, B != kByEntry> R;
  __shared__ __align__(16) float lds[kUpWaves][R::kFloats];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const Block blk = block_of(g, blockIdx.x, g.up_cols);
  const Ranks ranks(g);
  constexpr int kShare = PLAN ? 1 : kUpWaves;  // waves a group
  const int blocks = g.up_cols / kUpBlock, per = (blocks + kShare - 1) / kShare, first = wave % kShare * per;
  const int c0 = blk.c0 + kUpBlock * first, c1 = min(blk.c0 + kUpBlock * min(first + per, blocks), blk.end);
  for (int64_t at = PLAN ? (int64_t)blockIdx.y * kUpWaves + wave : blockIdx.y; at < g.groups;
       at += (int64_t)gridDim.y * (PLAN ? kUpWaves : 1)) {
    const Group gr = PLAN ? group_by_plan(g, at) : group_by_ballot(g, at);
    if (gr.count <= 0) continue;
    if (c0 >= c1) continue;
    const int live = ranks.of(g, gr.slot);
    if (!live && g.base == g.out) continue;
    R rows(g, gr, c0, blk.end);
    rows.load();
    if (!live) {
      for (int c = c0;;) {
        rows.copy();
        if (ONE || (c += kUpBlock) >= c1) break;
        rows.advance();
        rows.load();
      }
      continue;
    }
    TOperand<XT, NB, PACK, S> t;
    t.load(g, gr.row, blk.part);
    Columns<XT, NB, PACK, B> columns(g, gr.slot, c0, blk.end, live);
    vec8<XT> b[kUpTiles][NB];
#pragma unroll
    for (int n = 0; n < kUpTiles; ++n) columns.next(b[n]);
    for (int c = c0;;) {
      rows.add([&](int n) { return up_mma(b[n], t); }, lds[wave]);
      if (ONE || (c += kUpBlock) >= c1) break;
      rows.advance();
      rows.load();
#pragma unroll
      for (int n = 0; n < kUpTiles; ++n) columns.next(b[n]);
    }
  }
}

// ---- both in one launch ----------------------------------------------------------------------

constexpr int kOneStages = 2, kOneWaves = 8, kOneTiles = kLoraFusedCols / (16 * kOneWaves);

// Grid: (column blocks, rows).  The workgroup's waves share K of the first product, for its partition's rows of A alone, and
// meet in LDS; then each multiplies its own columns.
template <typename XT, int NB, bool PACK, int B>
__global__ __launch_bounds__(64 * kOneWaves) void lora_one_kernel(LoraArgs g) {
  constexpr int NT = kOneTiles, T = kBlockTiles<PACK>, N = T * NB;  // 16-row tiles of A
  constexpr bool VEC = B != kByEntry;
  typedef Rows<XT, NT, VEC> R;
  // A wave's stages; then its sums, later its result, in the first 4 KiB, and in the first wave's the parts of t past them.
  constexpr int kPartsBytes = NB * 16 * kBlockBytes<XT, PACK>, kUsed = 4096 + kPartsBytes + NB * 64;
  constexpr int kPitch = (std::max(VEC ? kDownBytes<N, kOneStages> : 0, kUsed) + 1023) & ~1023;
  static_assert(1024 * N <= 4096 && 4 * R::kFloats <= 4096, "the sums and the result");
  __shared__ __align__(1024) uint8_t stages[kOneWaves][kPitch];
  typedef uint8_t TBlock[kBlockBytes<XT, PACK>];
  TBlock(*blocks)[16] = (TBlock(*)[16])(stages[0] + 4096);  // [NB][16]
  int(*exps)[16] = (int(*)[16])(stages[0] + 4096 + kPartsBytes);
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const Block blk = block_of(g, blockIdx.x, kLoraFusedCols);
  const int c0 = blk.c0 + 16 * NT * wave, tok = lane & 15;
  const Ranks ranks(g);
  const int steps = (g.k + 31) >> 5, per = ((steps + kOneWaves - 1) / kOneWaves + 1) & ~1;
  const int s0 = min(wave * per, (steps + 1) & ~1), s1 = min(s0 + per, steps);
  for (int64_t at = blockIdx.y; at < g.groups; at += gridDim.y) {
    const Group gr = group_by_ballot(g, at);
    if (!gr.count) continue;
    const int live = ranks.of(g, gr.slot);
    if (!live && g.base == g.out) continue;
    R rows(g, gr, c0, blk.end);
    rows.load();
    if (!live) {
      rows.copy();
      continue;
    }
    Columns<XT, NB, PACK, B> columns(g, gr.slot, c0, blk.end, live);
    vec8<XT> b[NT][NB];
#pragma unroll
    for (int n = 0; n < NT; ++n) columns.next(b[n]);
    const float scaling = g.scaling[gr.slot];
    __builtin_amdgcn_sched_barrier(0);  // in flight before the ring
    f32x4_t acc[N];
#pragma unroll
    for (int i = 0; i < N; ++i) acc[i] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
    auto row = [&](int i, int j) { return 16 * i + j < live ? 16 * i + j : 0; };
    down_steps<XT, N, kOneStages, VEC>(g, gr, (const XT*)g.a + ((int64_t)gr.slot * g.parts.count + blk.part) * g.rank * g.k,
                                       row, s0, s1, stages[wave], acc);
#pragma unroll
    for (int i = 0; i < N; ++i) ((f32x4_t*)stages[wave])[64 * i + lane] = acc[i];
    __syncthreads();
    if (wave < NB) {
      f32x4_t v[T];
      meet_waves<kOneWaves, T>(stages[0], kPitch, T * wave, 16 * T * wave, live, scaling, v);
      const int exp = scale_block<XT, T>(v);
      uint8_t* to = &blocks[wave][tok][8 * (lane >> 4)];
#pragma unroll
      for (int t = 0; t < T; ++t) store_parts<XT, PACK>(v[t], to + 32 * t);
      if (std::is_same<XT, f16_t>::value && lane < 16) exps[wave][tok] = exp;
    }
    __syncthreads();  // (the sums are read: the result may take their place)
    TOperand<XT, NB, PACK> t;
#pragma unroll
    for (int k = 0; k < NB; ++k) {
#pragma unroll
      for (int h = 0; h < kOperands<XT, PACK>; ++h) t.v[k][h] = load_part<PACK>(blocks[k][tok], h);
      if constexpr (std::is_same<XT, f16_t>::value) t.exp[k] = exps[k][tok];
    }
    rows.add([&](int n) { return up_mma(b[n], t); }, (float*)stages[wave]);
    __syncthreads();  // before the next group's stages and parts
  }
}

// ---- the plan --------------------------------------------------------------------------------

constexpr int kPlanThreads = 1024, kPlanWaves = kPlanThreads / 64;

// 64 rows, one a lane: the lane's slot (slots: no adapter), and the lanes with the same one.
struct Window {
  bool in;
  int slot;
  uint64_t same;
  __device__ __forceinline__ Window(const int32_t* index, int64_t m, int slots, int64_t first) {
    const int lane = threadIdx.x & 63;
    in = first + lane < m;
    slot = in ? index[first + lane] : -1;
    if (slot < 0 || slot >= slots) slot = slots;
    same = same_slot(slot, slots, in);
  }
  __device__ __forceinline__ int before() const { return __popcll(same & ((1ull << (threadIdx.x & 63)) - 1)); }
  __device__ __forceinline__ bool leads() const { return in && before() == 0; }
};

// A stable counting sort by slot in one workgroup (bound by its six barriers: 100 rows 4.5 us, 2048 6.2, 65536 75; a step makes
// one plan for all of its linears): each wave counts a run of rows, the counts become first places, slot by
// slot and wave by wave, and the waves place their rows.
__global__ __launch_bounds__(kPlanThreads) void lora_plan_kernel(const int32_t* __restrict__ index, int64_t m, int slots,
                                                                 int32_t* __restrict__ plan) {
  extern __shared__ int32_t lds[];  // [kPlanWaves][slots + 1] counts, then places; [slots + 1] rows, first groups
  const int n = slots + 1, tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  int32_t *rows = lds + kPlanWaves * n, *first_group = rows + n;
  for (int i = tid; i < kPlanWaves * n; i += kPlanThreads) lds[i] = 0;
  __syncthreads();
  const int64_t run = (m + 64 * kPlanWaves - 1) / (64 * kPlanWaves) * 64;
  const int64_t r0 = wave * run, r1 = r0 + run < m ? r0 + run : m;
  int32_t* mine = lds + wave * n;
  for (int64_t r = r0; r < r1; r += 64) {
    const Window w(index, m, slots, r);
    if (w.leads()) mine[w.slot] += __popcll(w.same);  // one lane a slot
  }
  __syncthreads();
  for (int s = tid; s < n; s += kPlanThreads) {
    int total = 0;
    for (int w = 0; w < kPlanWaves; ++w) total += lds[w * n + s];
    rows[s] = total;
  }
  __syncthreads();
  if (wave == 0) {  // exclusive sums over the slots
    int groups = 0;
    for (int s0 = 0; s0 < n; s0 += 64) {
      const int t = s0 + lane < n ? (rows[s0 + lane] + kPlanGroup - 1) / kPlanGroup : 0;
      int ts = t;
#pragma unroll
      for (int o = 1; o < 64; o <<= 1) {
        const int tu = __shfl_up(ts, o, 64);
        if (lane >= o) ts += tu;
      }
      if (s0 + lane < n) first_group[s0 + lane] = groups + ts - t;
      groups += __shfl(ts, 63, 64);
    }
    if (lane == 0) plan[0] = groups, plan[1] = (int32_t)m, plan[2] = slots;
  }
  __syncthreads();
  for (int s = wave; s < n; s += kPlanWaves) {
    const int total = rows[s], first = first_group[s];
    for (int i = lane; i * kPlanGroup < total; i += 64)
      *(i32x2_t*)(plan + 4 + 2 * (int64_t)(first + i)) = i32x2_t{s < slots ? s : -1, min(kPlanGroup, total - i * kPlanGroup)};
  }
  for (int s = tid; s < n; s += kPlanThreads) {
    int place = first_group[s] * kPlanGroup;
    for (int w = 0; w < kPlanWaves; ++w) {
      const int c = lds[w * n + s];
      lds[w * n + s] = place;
      place += c;
    }
  }
  __syncthreads();
  int32_t* order = plan + plan_order_at(m, slots);
  for (int64_t r = r0; r < r1; r += 64) {
    const Window w(index, m, slots, r);
    const int place = mine[w.slot];
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");  // every lane has read its slot's place
    if (w.leads()) mine[w.slot] = place + __popcll(w.same);
    if (w.in) order[place + w.before()] = (int32_t)(r + lane);
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  }
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
  else if (rank <= 64) f(integral_constant<int, 2>{}, std::false_type{});
  else if (rank <= 96) f(integral_constant<int, 3>{}, std::false_type{});
  else f(integral_constant<int, 4>{}, std::false_type{});
}

template <typename F> void by_bool(bool v, F&& f) {
  if (v) f(std::true_type{});
  else f(std::false_type{});
}

template <typename F> void by_kind(int b, F&& f) {
  if (b == kAligned) f(std::integral_constant<int, kAligned>{});
  else if (b == kAnywhere) f(std::integral_constant<int, kAnywhere>{});
  else f(std::integral_constant<int, kByEntry>{});
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
  // The operands of each product as 16-byte vectors: x's, A's, base's and out's rows start on 16 bytes and K and the partitions are
  // multiples of 8; B's rows start anywhere, but a slot's B has 32-bit offsets, and 16 bytes at the least.
  const bool vec_k = g.k % 8 == 0 && aligned(g.x, g.ldx) && aligned(g.a, 0);
  const int64_t slot_b = (int64_t)g.n * g.rank;
  bool vec_n = aligned(g.base, g.ldb) && aligned(g.out, g.ldo) && slot_b >= 8 && slot_b < (1 << 30);
  for (int p = 0; p < g.parts.count; ++p) vec_n = vec_n && g.parts.end[p] % 8 == 0;
  const int b_kind = !vec_n ? kByEntry : g.rank % 8 == 0 && aligned(g.b, 0) ? kAligned : kAnywhere;
  const int chunks = cut_columns(g.parts, kLoraFusedCols);
  g.groups = lora_groups(g.m, g.slots);
  int reads = 0;
  for (int p = 0; p < g.parts.count; ++p) reads += std::min(8, g.parts.chunk_end[p] - (p ? g.parts.chunk_end[p - 1] : 0));
  if (lora_one_launch(g.plan, g.m, g.k, g.rank, g.slots, chunks, reads)) {
    by_rank(g.rank, [&](auto nb, auto pack) {
      if constexpr (32 * nb.value <= kLoraOneRank)
        by_kind(vec_k ? b_kind : kByEntry, [&](auto v) {
          qtts::launch(&lora_one_kernel<XT, nb.value, pack.value, v.value>, dim3(chunks, grid_y(g.groups)), dim3(64 * kOneWaves), 0,
                       st, g);
        });
    });
    return;
  }
  if (g.plan) g.groups = plan_max_groups(g.m, g.slots);
  const int a_tiles = g.parts.count * g.blocks * (g.rank <= 16 ? 1 : 2);
  const int down_tiles = lora_down_tiles(g.groups, a_tiles, g.rank <= 16), down_wide = (a_tiles + down_tiles - 1) / down_tiles;
  g.splits = vec_k && b_kind == kAligned ? lora_splits(g.m, g.k, g.rank, g.groups * down_wide) : 1;
  by_bool(g.plan, [&](auto plan) {
    by_bool(g.rank <= 16, [&](auto pack) {
      by_bool(vec_k, [&](auto v) {
        auto down = [&](auto n) {
          qtts::launch(&lora_down_kernel<XT, n.value, pack.value, v.value, plan.value>,
                       dim3(down_wide, grid_y(g.groups), g.splits), dim3(64 * kDownWaves), 0, st, g);
        };
        using std::integral_constant;
        if constexpr (pack.value) {
          if (down_tiles == 1) return down(integral_constant<int, 1>{});
          if (down_tiles == 3) return down(integral_constant<int, 3>{});
        }
        if (down_tiles == 2) down(integral_constant<int, 2>{});
        else down(integral_constant<int, 4>{});
      });
    });
    g.up_cols = lora_up_cols(g.m, g.n);
    const int up_chunks = cut_columns(g.parts, g.up_cols);
    by_rank(g.rank, [&](auto nb, auto pack) {
      by_kind(b_kind, [&](auto v) {
        auto launch_up = [&](auto s, auto one) {
          qtts::launch(&lora_up_kernel<XT, nb.value, pack.value, v.value, plan.value, s.value, one.value>,
                       dim3(up_chunks, grid_y(plan.value ? (g.groups + kUpWaves - 1) / kUpWaves : g.groups)),
                       dim3(64 * kUpWaves), 0, st, g);
        };
        auto up = [&](auto s) {
          if constexpr (plan.value && v.value == kAligned) {
            if (g.up_cols == kUpBlock) return launch_up(s, std::true_type{});
          }
          launch_up(s, std::false_type{});
        };
        if constexpr (v.value == kAligned && 32 * nb.value <= kLoraSplitRank) {
          if (g.splits == 2) return up(std::integral_constant<int, 2>{});
        }
        up(std::integral_constant<int, 1>{});
      });
    });
  });
}

}  // namespace

// The workspace: t's blocks, split by split and row by row, then fp16's exponents.
static int64_t lora_t_blocks(int64_t m, int64_t parts, int64_t rank) { return lora_max_splits(m, rank) * m * parts * lora_blocks(rank); }
static int64_t lora_t_bytes(int64_t m, int64_t parts, int64_t rank) {
  return align256(lora_t_blocks(m, parts, rank) * (rank <= 16 ? kBlockBytes<bf16_t, true> : kBlockBytes<bf16_t, false>));
}

int64_t qtts_lora_ws_bytes(int64_t m, int64_t parts, int64_t rank) {
  return kCounterBytes + lora_t_bytes(m, parts, rank) + align256(lora_t_blocks(m, parts, rank) * 4);
}

int qtts_launch_lora_plan(const int32_t* index, int64_t m, int64_t slots, int32_t* plan, hipStream_t st) {
  const uint32_t shmem = (uint32_t)((kPlanWaves + 2) * (slots + 1) * 4);
  qtts::launch(&lora_plan_kernel, dim3(1), dim3(kPlanThreads), shmem, st, index, m, slots, plan);
  return qtts_check_launch("lora_plan");
}

int qtts_launch_lora_add(const LoraArgs& args, int x_dtype, void* ws, hipStream_t st) {
  LoraArgs g = args;
  g.t = (uint8_t*)ws + kCounterBytes;
  g.exps = (int32_t*)(g.t + lora_t_bytes(g.m, g.parts.count, g.rank));
  g.blocks = lora_blocks(g.rank);
  if (x_dtype == QTTS_BF16) launch_lora<bf16_t>(g, st);
  else launch_lora<f16_t>(g, st);
  return qtts_check_launch("lora_add");
}
