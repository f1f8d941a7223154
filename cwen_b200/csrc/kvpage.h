// Page-table arithmetic of the paged cache, for the kernels and the host.
//
// A cache pool is [layer][page][slot in the page][kv head][head_dim]; a
// sequence's table row holds the page ids of its slots in order.  Page ids
// come from device memory that the host cannot check, so every lookup is
// checked here and a bad one gives -1: nothing outside the pool is touched.
#pragma once
#include <stdint.h>

#ifdef __CUDACC__
#define CWP_FN __host__ __device__ __forceinline__
#else
#define CWP_FN static inline
#endif

// Place in a sequence's table row of the page that holds `slot`, or -1.
CWP_FN int64_t cwp_entry(int table_stride, int page_size, int64_t slot) {
  if (slot < 0 || slot >= (int64_t)table_stride * page_size) return -1;
  // in range, slot / page_size < table_stride: 32-bit arithmetic where it can be
  return slot <= 0x7fffffff ? (int64_t)((uint32_t)slot / (uint32_t)page_size) : slot / page_size;
}
// Pool row of `slot` whose table entry (at cwp_entry) is `page`, or -1 when that is no page of the pool.
CWP_FN int64_t cwp_row_in(int page, int64_t entry, int n_pages, int page_size, int64_t slot) {
  if (page < 0 || page >= n_pages) return -1;
  return (int64_t)page * page_size + (slot - entry * page_size);
}
// Pool row (page * page_size + slot in the page) of a sequence's `slot`, or
// -1 when the slot lies outside the table row or its page id outside
// [0, n_pages).  64 bits: a pool may hold more than 2^31 rows' elements.
CWP_FN int64_t cwp_row(const int *table_row, int table_stride, int n_pages, int page_size, int64_t slot) {
  const int64_t e = cwp_entry(table_stride, page_size, slot);
  return e < 0 ? -1 : cwp_row_in(table_row[e], e, n_pages, page_size, slot);
}
