// Index arithmetic of the paged key/value cache and of the ragged batch that
// uses it.  Plain C++ on values (no device types), so that a host program can
// compile it and check every case that a caller's device arrays can hold: the
// host does not see them, so the kernels bound each entry before it becomes an
// address.
#pragma once

#include <stdint.h>

#ifdef __HIP__
#define MOE_HD __host__ __device__ __forceinline__
#else
#define MOE_HD inline
#endif

namespace moe {

// Rows [first, first + rows) of the batch are the new tokens of a sequence
// whose cached length, the new tokens included, is len.  Row first + i is at
// position base + i; base < 0 when len < rows, and rows at a negative position
// have no place in the cache.
struct SeqSpan {
  int32_t first, rows, len, base;
  bool ok;   // every entry inside its range
};

// start, end: the sequence's entries of the row starts; total: the batch's
// rows; cap: positions that its row of the page table covers.
MOE_HD SeqSpan seq_span(int32_t start, int32_t end, int32_t len, int32_t total, int32_t cap) {
  SeqSpan s;
  const int32_t a = start < 0 ? 0 : start > total ? total : start;
  const int32_t b = end < a ? a : end > total ? total : end;
  const int32_t n = len < 0 ? 0 : len > cap ? cap : len;
  s.first = a;
  s.rows = b - a;
  s.len = n;
  s.base = n - s.rows;
  s.ok = a == start && b == end && n == len && s.base >= 0;
  return s;
}

// Element offset of position `pos` (inside a sequence's table row) for one key
// head in pages laid out [n_pages, heads, page, dim], or -1 where the table
// entry names no page.
MOE_HD int64_t page_row(int32_t entry, int32_t n_pages, int32_t heads, int32_t head,
                        int32_t page_shift, int32_t pos, int32_t dim) {
  if (entry < 0 || entry >= n_pages) return -1;
  const int64_t row = (((int64_t)entry * heads + head) << page_shift) +
                      (pos & ((1 << page_shift) - 1));
  return row * dim;
}

// Keys [lo, hi) that a row at position pos sees in a sequence of n cached
// tokens: all up to its own, or the last `window` of those (window > 0).
// Empty for a negative position.
MOE_HD void seen_keys(int32_t pos, int32_t n, int32_t window, int32_t *lo, int32_t *hi) {
  *hi = pos < 0 ? 0 : pos < n ? pos + 1 : n;
  *lo = window > 0 && pos >= window ? pos - window + 1 : 0;
}

}  // namespace moe
