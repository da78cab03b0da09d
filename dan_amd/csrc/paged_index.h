// Where a place of a sequence lies in a paged cache (device code, and host code for its test).
#pragma once
#include <stdint.h>

#ifdef __HIPCC__
#define DAN_INDEX_FN __host__ __device__ inline
#else
#define DAN_INDEX_FN inline
#endif

namespace dan {

struct PageTable {
  const int32_t *pages;    // [seqs, width]
  int64_t stride;          // of a row
  int32_t seqs, width;
  int32_t page_size;       // rows of a page
  int32_t num_pages;       // of the cache
};

struct PageRow {
  int32_t page;  // in [0, num_pages), or -1: nothing may be read or written there
  int32_t row;   // in [0, page_size)
};

// Nothing the device holds is trusted: a sequence, a place or a page that does not exist
// gives page -1, and the table is read inside its bounds only.
DAN_INDEX_FN PageRow find_row(const PageTable &t, int32_t seq, int32_t place) {
  if (place < 0 || (uint32_t)seq >= (uint32_t)t.seqs) return {-1, 0};
  const uint32_t nth = (uint32_t)place / (uint32_t)t.page_size;
  if (nth >= (uint32_t)t.width) return {-1, 0};
  const int32_t page = t.pages[seq * t.stride + nth];
  if ((uint32_t)page >= (uint32_t)t.num_pages) return {-1, 0};
  return {page, (int32_t)((uint32_t)place - nth * (uint32_t)t.page_size)};
}

}  // namespace dan
