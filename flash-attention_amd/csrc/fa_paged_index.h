// Arithmetic on what lies in device memory and is not trusted with an address: plain C++, so that its limits can be tested on a host.
#pragma once

#include <cstdint>

#if defined(__HIP__)
#define FA_INDEX __host__ __device__ __forceinline__
#else
#define FA_INDEX inline
#endif

namespace fa {

// A page table entry as it is read: a page of the pool whatever it holds.
FA_INDEX int page_in_pool(int page, int n_pages) { return page < 0 ? 0 : (page < n_pages ? page : n_pages - 1); }
// ... as it is written to: only if it is one.
FA_INDEX bool page_is_one(int page, int n_pages) { return page >= 0 && page < n_pages; }
// A sequence's length: at most what the table holds and the caller said.
FA_INDEX int keys_in_reach(int len, int max_keys) { return len < 0 ? 0 : (len < max_keys ? len : max_keys); }
// The slot of packed row `row` of a sequence that ends before row `end` and then has `len` keys; -1: none.  begin, end: the sequence's rows
FA_INDEX int append_slot(int len, int begin, int end, int row, int max_rows, int max_keys) {
  const int64_t slot = (int64_t)len - ((int64_t)end - row);
  const bool ok = (begin >= 0) & (row >= begin) & (row < end) & ((int64_t)end - begin <= max_rows) & (slot >= 0) & (slot < max_keys);
  return ok ? (int)slot : -1;  // (no branches: a wave looks at several rows at once)
}
// A table row for a position: the nearest one.
FA_INDEX int table_row(int pos, int rows) { return pos < 0 ? 0 : (pos < rows ? pos : rows - 1); }

}  // namespace fa
