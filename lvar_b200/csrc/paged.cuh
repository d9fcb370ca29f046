// The paged key/value cache as the kernels see it: pages [num_pages, Hkv, page_size, D] of bf16, or of e4m3 with one
// power-of-two scale per row, and per sequence a row of page numbers.
#pragma once

#include "common.cuh"

namespace lvar {

// Strides in BYTES.  Rows of a page are addressed by groups of 16, which never cross a page.
struct PagedView {
  uint8_t* k;
  uint8_t* v;
  uint8_t* scales;  // biased exponents (2^(x - 127)) [num_pages, Hkv, page_size, 2]: K's and V's; null: bf16 cache
  int64_t k_sp, k_sh, k_sl;
  int64_t v_sp, v_sh, v_sl;
  int64_t s_sp, s_sh;
  const int32_t* table;
  int64_t t_sb;  // entries
  int32_t num_pages, max_pages;
  uint32_t groups;  // 16-row groups per page
  uint32_t magic;   // ceil(2^32 / groups); 0 for one group per page
};

// Page index of a sequence's 16-row group n < 2^27: exact, since magic * groups - 2^32 < groups <= 32 and so
// n * (magic * groups - 2^32) < 2^32.
__device__ __forceinline__ uint32_t page_of_group(const PagedView& c, uint32_t n) {
  return c.magic ? __umulhi(n, c.magic) : n;
}

// Checks a cache description and fills the view.  Returns an LVAR_* code.
int paged_view(const lvar_paged_cache* c, PagedView* out);

}  // namespace lvar
