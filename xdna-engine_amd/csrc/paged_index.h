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
// stream -- lie in a row, [0, total), and workgroup i takes [i * per, (i + 1) *
// per): equal shares, from the middle of one unit to the middle of another.
XE_HD unsigned share_of(unsigned total, unsigned workgroups) { return (total + workgroups - 1) / workgroups; }

// Whole quotients by a divisor that is used often: m = floor((2^32 - 1) / d)
// gives floor(n / d) or one less.
struct Div {
  unsigned d, m;
};
XE_HD Div div_by(unsigned d) { return Div{d, 0xffffffffu / d}; }
XE_HD unsigned quot(unsigned n, const Div &v) {
  const unsigned q = static_cast<unsigned>((static_cast<unsigned long long>(n) * v.m) >> 32);
  return q + (n - q * v.d >= v.d ? 1u : 0u);
}
XE_HD unsigned quot_up(unsigned n, const Div &v) {
  const unsigned q = quot(n, v);
  return q + (q * v.d != n ? 1u : 0u);
}

// Whole workgroups a unit: workgroup i of the `wgs` that share a unit of n
// granules takes [t0, t1), as equal as can be.
XE_HD void part_of(unsigned n, unsigned wgs, unsigned i, unsigned &t0, unsigned &t1) {
  const unsigned q = n / wgs, r = n - q * wgs;
  t0 = q * i + (i < r ? i : r);
  t1 = t0 + q + (i < r ? 1u : 0u);
}
// Granules a workgroup takes at least, so that units of up to `alone` stay in
// one and the longest needs no second level of groups of partials where `more`
// a workgroup avoid it.
XE_HD unsigned least_share(unsigned longest, unsigned group, unsigned alone, unsigned more) {
  if (longest <= alone) return longest;
  const unsigned q = (longest + group - 1) / group;
  return q <= more ? (q < more / 3 ? more / 3 : q) : 1;
}

// Whether units get whole workgroups, else equal shares: up to 64 streams (a lane
// of a wave each) of up to a unit a CU, of fewer than kManyUnits units or of keys
// (`span` a unit: what the table or the window allows) up to kFewBytes.  us in
// whole workgroups / in shares: 32768 keys of one stream (4 x 256) 18.2 / 23.6, 8
// mixed streams to 3000 keys (8 / 2 x 128) 9.7 / 10.8, 32 of window 1024 12.5 /
// 16.5, 60 to 300 keys (16 / 4 x 128) 9.4 / 13.6, 64 to 1500 (4 x 256) 20.9 / 26.5,
// 64 to 4096 50.3 / 46.1.  8, 16, 32, 48 and 63 streams of one length (4 / 1 x 256):
//    64 MB   22.0 / 25.6  19.2 / 26.6  19.4 / 24.8  19.7 / 23.6  19.6 / 25.5
//   150 MB   34.0 / 39.6  32.0 / 39.0  32.2 / 35.9  32.9 / 36.4  33.2 / 37.0
//   300 MB   62.1 / 59.7  59.2 / 61.6  59.4 / 59.7  60.0 / 58.8  59.9 / 59.7
//   500 MB   95.8 / 88.6  93.1 / 89.4  93.5 / 89.8  92.7 / 87.6  93.3 / 88.0
// (mixed lengths and 8 / 2 and 32 / 8 x 128 alike): by bytes the two meet at about
// 250 MB, and fewer than kManyUnits units beyond that are up to 8 % slower so.
constexpr int kManyUnits = 64;
constexpr int64_t kFewBytes = int64_t(128) << 20;
inline bool whole_units(int batch, int64_t units, int64_t span, int hd, int cus) {
  return batch <= 64 && units <= cus && (units < kManyUnits || units * span * hd * 4 <= kFewBytes);
}

// Shares begin at i * per, or at the end of a unit that lies at most `slack`
// granules from there: neither a unit of few granules nor an end of one is
// split off for its sake.  g lies in a unit of n granules of the stream that
// begins at granule base.
XE_HD unsigned snapped(unsigned g, unsigned base, unsigned n, unsigned slack) {
  const unsigned off = (g - base) % n;
  return off <= slack && off <= n - off ? g - off : n - off <= slack ? g - off + n : g;
}
// Workgroups that the unit of granules [u0, u0 + n) is spread over: wgs of
// them, from w0 on (wgs = 1: the one whose share it lies in, w0 is not set).
XE_HD void spread(unsigned u0, unsigned n, const Div &per, unsigned slack, unsigned &w0, unsigned &wgs) {
  wgs = 1;
  if (n <= 2 * slack) return;
  // shares that begin within it, further than slack from its ends
  const unsigned a = quot(u0 + slack, per) + 1, z = quot(u0 + n - slack - 1, per);
  if (z < a) return;
  w0 = a - 1;
  wgs = z - a + 2;
}

// Place of workgroup wg's partial of the unit that begins at granule u0: a
// workgroup has at most one unit that began before it and one that it begins
// and does not end.
XE_HD unsigned slot_of(unsigned u0, unsigned per, unsigned wg) { return 2 * wg + (u0 >= wg * per ? 1u : 0u); }

}  // namespace paged
}  // namespace xe
