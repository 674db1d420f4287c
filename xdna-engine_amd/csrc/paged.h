// paged.h -- launch surface of the paged KV cache (paged_append.hip,
// paged_attn.hip) and of the int8 linears with a scale a row (rows_q8.hip).
#pragma once

#include "common.h"
#include "paged_index.h"

namespace xe {

struct PagedView {
  uint16_t *k = nullptr, *v = nullptr;
  const int32_t *table = nullptr;  // [batch, max_pages]
  size_t page_stride = 0;          // elements from page to page
  int n_pages = 0, page_shift = 0, hkv = 0, hd = 0, batch = 0, max_pages = 0;
};
// Checks kv (xe_paged_kv) and gives its view.
PagedView paged_view(const xe_paged_kv *kv);

void launch_paged_append(const PagedView &kv, const xe_paged_rows &r, hipStream_t s);

struct PagedAttn {
  PagedView kv;
  const float *q = nullptr;
  size_t ldq = 0;
  const int32_t *lens = nullptr;
  int hq = 0;
  float scale = 1.0f;
  int window = 0;
  float *out = nullptr;
  size_t ldo = 0;
};
// work / cnt: partials of units that several workgroups share
// (paged_work_floats()) and arrival counters (paged_cnt_words(), zeroed once;
// they re-arm).
void launch_paged_attn(const PagedAttn &a, float *work, unsigned *cnt, hipStream_t s);
size_t paged_work_floats();
size_t paged_cnt_words();

// y = act((q . w) s ws + bias) + res over the int8 codes q of norm(x + add)
// and their row scales s; codes / scales: workspace, rows_q8_codes_bytes() and
// batch floats.  kp, vec: set by the launch (a row of codes with its padding,
// whether results of four weight rows go out at once).
struct RowsQ8 {
  const int8_t *w = nullptr;
  const float *ws = nullptr, *bias = nullptr;
  int m = 0, k = 0, norm = XE_NORM_NONE;
  const float *gamma = nullptr, *beta = nullptr;
  float eps = 0.f;
  xe_w8a8_rows a{};
  int8_t *codes = nullptr;
  float *scales = nullptr;
  int *part = nullptr;
  unsigned *cnt = nullptr;
  int kp = 0, vec = 0;
};
size_t rows_q8_codes_bytes(int batch, int k);
// Scales (2 KB), then arrival counters (4 KB, zeroed once; they re-arm), then
// partial tiles of K splits.
size_t rows_q8_ws_bytes();
int launch_rows_q8(const RowsQ8 &r, hipStream_t s);  // returns its launches

}  // namespace xe
