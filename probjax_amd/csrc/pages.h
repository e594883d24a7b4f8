// A paged KV cache as the kernels take it (paged_cache.hip, paged_decode.hip): pools
// of pages for K and V, a row of page numbers per sequence, and in 8 bits a power of
// two per row (one token's key or value of one head).
#pragma once

#include <type_traits>

#include "pjx_common.h"
#include "pjx_internal.h"

namespace pjx {

// Division of 0 <= n < 2^31 by d: n * ceil(2^(31+s) / d) / 2^(31+s), 2^s >= d, exact
// over that range; the multiplier fits 32 bits, one more than the product's shift needs.
struct FastDiv {
  uint32_t mul;
  int shift;
  __device__ __forceinline__ int operator()(int n) const { return (int)(__umulhi(2u * (uint32_t)n, mul) >> shift); }
};
inline FastDiv fast_div(int64_t d) {
  int s = 0;
  while (((int64_t)1 << s) < d) ++s;
  const unsigned __int128 one = (unsigned __int128)1 << (31 + s);
  return {(uint32_t)((one + d - 1) / d), s};
}

struct PageArgs {
  char *k, *v;        // pools
  uint8_t *ke, *ve;   // [pages][H][page] exponent + 127 of every row, or null
  const int32_t* table;
  int64_t table_step;  // entries between sequences
  uint32_t pages;
  int page, most;      // slots of a page, pages of a sequence
  int H;
  FastDiv by_page;
  int64_t kp, kt, kh, vp, vt, vh;  // bytes between pages, tokens and heads of the pools
};

// Page i < most of sequence b, as the table has it; no page unless below a.pages.
__device__ __forceinline__ uint32_t page_entry(const PageArgs& a, int b, int i) {
  return a.table ? (uint32_t)a.table[b * a.table_step + i] : (uint32_t)b;
}

// Float formats beside Bf16Fmt and F16Fmt, and the format of 8-bit caches.
struct F32Fmt {};
struct E4m3Fmt {};
template <typename F>
constexpr int fmt_size() {
  return std::is_same<F, F32Fmt>::value ? 4 : std::is_same<F, E4m3Fmt>::value ? 1 : 2;
}

__device__ __forceinline__ float exponent_scale(uint32_t e) { return __uint_as_float(e << 23); }

// Checks a pjx_pages (paged_cache.hip) and fills `a`; a PJX_* status.
int fill_pages(PageArgs& a, const char* who, int cache_dtype, const pjx_pages* cache, int64_t batch, int64_t kv_heads,
               int64_t head_dim);

}  // namespace pjx
