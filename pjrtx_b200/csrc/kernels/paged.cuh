// Device-side view of a paged key-value cache.
#pragma once

#include "operators.h"

namespace pjrtx {

// Reports an argument that only the device sees. A word for each code, so that none replaces another; every writer writes the same.
__device__ __forceinline__ void report(int* error_words, int code) {
  *const_cast<volatile int*>(error_words + (code - kErrorPageId)) = 1;
}

// Visible rows of a sequence, held to what its page table can name.
__device__ __forceinline__ int paged_length(const PagedView& c, int b) {
  const int n = c.lengths[b];
  const int capacity = c.page_size * c.max_pages;
  return n < 0 ? 0 : n > capacity ? capacity : n;
}

// Whether the length itself is in range (asked by one thread of one block per sequence).
__device__ __forceinline__ void paged_check_length(const PagedView& c, int b) {
  const int n = c.lengths[b];
  if (n < 0 || n > c.page_size * c.max_pages) report(c.error_words, kErrorLength);
}

// Element offset of row `slot` of sequence b in either pool (KV head 0), or -1 where the table names no page.
__device__ __forceinline__ long long paged_row(const PagedView& c, int b, int slot) {
  const int column = slot / c.page_size;
  const int page = c.table[b * c.table_stride + column];
  if (page < 0 || page >= c.num_pages) {
    report(c.error_words, kErrorPageId);
    return -1;
  }
  return page * c.page_stride + (long long)(slot - column * c.page_size) * c.row_stride;
}

}  // namespace pjrtx
