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

// Attention's work is counted in granules of kg keys (kg a power of two), the
// first of a stream at the last multiple of 16 at or before its first key.
XE_HD unsigned granules(int lo, int hi, int kg) {
  return hi > lo ? static_cast<unsigned>((hi - (lo & ~15) + (kg - 1)) / kg) : 0u;
}

// The granules of all units -- unit (stream, block of query heads), stream by
// stream -- in a row, [0, total), are shared out in equal ranges: workgroup i
// takes [i * per, (i + 1) * per).
XE_HD unsigned share_of(unsigned total, unsigned workgroups, unsigned least) {
  const unsigned per = (total + workgroups - 1) / workgroups;
  return per < least ? least : per;
}

// Workgroups that the unit of granules [u0, u1) is spread over: first_wg(u0)
// and the ones behind it.
XE_HD unsigned first_wg(unsigned u0, unsigned per) { return u0 / per; }
XE_HD unsigned wg_count(unsigned u0, unsigned u1, unsigned per) { return (u1 - 1) / per - u0 / per + 1; }

// Place of workgroup wg's partial of that unit: a workgroup has at most one
// unit that began before it and one that it begins and does not end.
XE_HD unsigned slot_of(unsigned u0, unsigned per, unsigned wg) { return 2 * wg + (u0 >= wg * per ? 1u : 0u); }

}  // namespace paged
}  // namespace xe
