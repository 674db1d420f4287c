// paged_index.h -- where a stream's keys lie in a paged cache: plain integer
// arithmetic of the paged kernels, also compiled for the host (its tests).
#pragma once

#include <cstddef>
#include <cstdint>

#ifdef __HIPCC__
#define XE_HD __host__ __device__ __forceinline__
#else
#define XE_HD inline
#endif

namespace xe {
namespace paged {

// Page of position pos of the stream whose table row is `row`, or -1: a
// position outside the table, or an entry that is no page.
XE_HD int page_of(const int32_t *row, int max_pages, int n_pages, int page_shift, long long pos) {
  if (pos < 0 || (pos >> page_shift) >= max_pages) return -1;
  const int p = row[pos >> page_shift];
  return p >= 0 && p < n_pages ? p : -1;
}

// Element offset of (page, kv head, slot) in K or V; may pass 32 bits.
XE_HD size_t row_at(size_t page_stride, int page_shift, int hd, int page, int head, int slot) {
  return static_cast<size_t>(page) * page_stride +
         ((static_cast<size_t>(head) << page_shift) + static_cast<size_t>(slot)) * static_cast<size_t>(hd);
}

// Keys [lo, hi) that the newest token of a stream of len tokens attends to:
// the last `window` of them (0: all), those past the table left out.
XE_HD void key_range(int len, int window, int capacity, int &lo, int &hi) {
  lo = window > 0 && len > window ? len - window : 0;
  hi = len < capacity ? len : capacity;
  if (hi < lo) hi = lo;
}

}  // namespace paged
}  // namespace xe
