// A paged key-value cache and what a step does with it (paged_step.hip, qkv_cache.hip, paged_attention.hip).
//
// The cache: pages of S = 2^page_shift tokens, k [pages, kv_heads, S, d] and v [pages, kv_heads, d, S] (d-major: eight
// consecutive tokens of one dimension are one 16-byte matrix operand of the second product).  Request r's tokens
// [j S, (j + 1) S) are on page table[r, j].  A slot is page * S + token on the page.
#pragma once

#include <stdint.h>

namespace qtts {

constexpr int kPagedMaxRequests = 2048;
constexpr int kPagedMinShift = 4, kPagedMaxShift = 10;  // pages of 16 to 1024 tokens
constexpr int kPagedMaxDim = 256;

struct PagedCache {
  void* k;
  void* v;
  int32_t pages, page_shift, kv_heads, d;
};

struct PagedStepArgs {
  const int32_t* added;  // [requests]
  const int32_t* lengths;
  int32_t* table;  // [requests, cols]
  const int32_t* free_pages;
  const int32_t* taken;
  int32_t* starts;  // [requests + 1]
  int32_t* counts;
  int32_t* lengths_out;  // may be lengths
  int32_t* taken_out;    // may be taken
  int32_t* positions;    // [rows]
  int32_t* slots;
  uint32_t* ticket;  // a zero counter, left at zero; used by grids of several workgroups
  int32_t requests, cols, pages, page_shift, rows, room, max_new;
};

struct QkvCacheArgs {
  const void* qkv;  // [rows, (heads + 2 kv_heads) d]
  int64_t ldqkv;
  const int32_t* positions;
  const int32_t* slots;
  const void* q_norm;  // [d] or null
  const void* k_norm;
  const float* cos;  // [rope_rows, d / 2] or null
  const float* sin;
  void* q;  // [rows, heads, d]
  PagedCache cache;
  int32_t rows, heads, rope_rows;
  float eps;
};

struct PagedAttentionArgs {
  const void* q;  // [rows, heads, d], row stride ldq
  int64_t ldq;
  void* out;
  int64_t ldo;
  const int32_t* table;  // [requests, cols]
  const int32_t* starts;
  const int32_t* counts;
  const int32_t* lengths;
  PagedCache cache;
  int32_t rows, heads, requests, cols, max_new, window, sinks;
  float scale;  // times log2 e
  bool weights16;  // the weights of runs of more than 16 rows in 16 bits
};

}  // namespace qtts
