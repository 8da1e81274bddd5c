// Where a token of an utterance lies in the paged cache: plain arithmetic, compiled for the kernels and, by the tests, for
// the host.
#pragma once

#include <stdint.h>

#ifdef __HIPCC__
#include <hip/hip_runtime.h>
#define TACO_HD __host__ __device__ __forceinline__
#else
#define TACO_HD inline
#endif

constexpr uint32_t TACO_KV_BAD_PAGE = 1, TACO_KV_BAD_PLACE = 2;   // bits of taco_kv_cache::flags
constexpr int32_t TACO_KV_MAX_TOKENS = 1 << 30;                   // of one utterance

// n / div for n < 2^30 by a multiplication (the divisor is a page's size, known when a kernel is launched): with
// L = floor(log2 div) and mul = floor(2^(31+L) / div) + 1 the product is too large by n * (mul * div - 2^(31+L)) / (div *
// 2^(31+L)) < 1 / div, because mul * div - 2^(31+L) <= div < 2^(L+1).
struct taco_divisor {
  uint32_t mul, shift, div;
};
inline taco_divisor taco_make_divisor(uint32_t d) {
  const uint32_t L = 31 - (uint32_t)__builtin_clz(d);
  return {(uint32_t)((1ull << (31 + L)) / d + 1), 31 + L, d};
}
TACO_HD uint32_t taco_divide(uint32_t n, const taco_divisor& f) { return (uint32_t)(((uint64_t)n * f.mul) >> f.shift); }

// A place in the cache: page < 0 where there is none, then `flag` says why.
struct taco_place {
  int32_t page;
  uint32_t unit;      // token (or block of tokens) inside the page
  uint32_t flag;
};
// Unit `at` of an utterance whose table row is `row`; a page holds per_page.div units.
TACO_HD taco_place taco_find(const int32_t* row, int32_t table_width, int32_t n_pages, int64_t at, const taco_divisor& per_page) {
  if (at < 0 || at >= TACO_KV_MAX_TOKENS) return {-1, 0, TACO_KV_BAD_PLACE};
  const uint32_t no = taco_divide((uint32_t)at, per_page);
  if (no >= (uint32_t)table_width) return {-1, 0, TACO_KV_BAD_PLACE};
  const int32_t page = row[no];
  if (page < 0 || page >= n_pages) return {-1, 0, TACO_KV_BAD_PAGE};
  return {page, (uint32_t)at - no * per_page.div, 0};
}
