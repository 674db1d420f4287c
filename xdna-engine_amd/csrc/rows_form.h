// rows_form.h -- on which way an int8 linear's rows become codes, and which form
// of the product a shape takes.
#pragma once

#include <cstddef>
#include <cstdint>

namespace xe {
namespace rowsform {

constexpr size_t kPartBytes = size_t(32) << 20;  // workspace of partial tiles
constexpr int kTiles = 1024;                     // tiles that have an arrival counter

// The forms and the time, in us, that each is estimated to take:
//   fixed + steps (step + round (rounds - 1)) + out m batch / 10^6
// with `steps` of K a workgroup and `rounds` of workgroups a CU.  Fitted to 534
// shapes (m 128 to 14336, K 768 to 14336, 2 to 512 rows), to 5 to 9 % a form.
// The form of the least estimate is 0.3 % slower than the fastest of all on
// average, 8 % at most.  Measured us of the forms in the order of the table (-:
// its partial tiles do not fit; .: not measured):
//   m x K        rows
//   512 x 14336     8     11   12   19   26   16   12   36    .    .  6.9  7.2
//   4096 x 4096    16    6.2  6.7  8.9   12   10   11   14   19   28   10  9.3
//   4096 x 4096    64     14  9.6  9.0   12   11   12   15   20   33   26   15
//   4096 x 14336   64     37   23   20   30   21   18   38   53   84   48   31
//   4096 x 14336  200    109   71   68   32   29   32   38   52   83    .    .
//   14336 x 4096  200    128   81   70   31   34    -   26   23   35    .    .
//   14336 x 4096  512    306  182  155   59    -    -   54   50   45    -    -
struct Form {
  int bm, bn;    // the tile: weight rows x activation rows
  int k;         // K a workgroup takes at once: 4 waves' 64 each, or all waves' 128
  int ksplit;    // workgroups that share K
  float fixed, step, round, out;
};
constexpr int kForms = 11;
constexpr Form kForm[kForms] = {
    {16, 16, 256, 1, 2.51f, 0.159f, 0.132f, 11.5f},   {16, 32, 256, 1, 2.60f, 0.186f, 0.172f, 4.22f},
    {32, 32, 256, 1, 2.88f, 0.301f, 0.285f, 3.11f},   {64, 64, 128, 1, 3.25f, 0.229f, 0.141f, 1.82f},
    {64, 64, 128, 2, 5.00f, 0.242f, 0.150f, 3.10f},   {64, 64, 128, 4, 6.37f, 0.279f, 0.175f, 4.66f},
    {128, 64, 128, 1, 3.44f, 0.305f, 0.219f, 1.72f},  {128, 128, 128, 1, 4.41f, 0.434f, 0.558f, 1.43f},
    {256, 128, 128, 1, 6.85f, 0.682f, 0.682f, 2.12f}, {16, 16, 256, 4, 4.28f, 0.185f, 0.139f, 49.2f},
    {16, 32, 256, 4, 4.28f, 0.230f, 0.188f, 21.2f}};

// Codes and product in one launch or in two; rows off 16 bytes, and results that
// lie over other workgroups' inputs, always take two.
// One row of K up to kFusedK: each workgroup makes the codes for itself, behind its
// first weight loads.  us in one launch / in two: 768 -> 768 4.4 / 6.2, 4096 ->
// 4096 7.4 / 9.0, 1152 -> 13824 7.5 / 10.6.  Two rows one after the other took
// longer than two launches where K is 4096.  32 weight rows a workgroup / 16: those
// 4.8 / 4.4, 8.9 / 7.4, 7.5 / 8.2; 2048 -> 9000 8.6 / 8.4.
// Up to kManyRows rows, a wave each, where that is one tile a CU.  us in one launch /
// in two, 2 and 8 rows: 768 -> 1536 5.4 / 6.8, 5.4 / 6.9, 1152 -> 4096 6.6 / 7.1,
// 6.6 / 7.4; 1600 -> 4096 7.6 / 7.1, 7.4 / 7.3; 16 rows on sixteen waves 768 ->
// 1536 7.0 / 6.4, 256 -> 1536 6.4 / 6.2; four tiles a CU, 1152 -> 13824, 20 / 8.8.
// One row so: 768 -> 1536 5.3, on all its workgroup's threads 4.6.
constexpr int kFusedK = 4096;
constexpr int kManyRows = 8, kManyK = 1280;
enum Way { kOneRow, kOneRowWide, kWaveRows, kTwoLaunches };
inline Way way(int m, int k, int batch, int cus) {
  if (batch == 1 && k <= kFusedK) return m > 32 * cus ? kOneRowWide : kOneRow;
  return batch <= kManyRows && m <= 16 * cus && k <= kManyK ? kWaveRows : kTwoLaunches;
}

inline int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

// Whether the partial tiles of form i have room in the workspace.
inline bool fits(int i, int m, int batch) {
  const Form &f = kForm[i];
  if (f.ksplit == 1) return true;
  const int64_t tiles = ceil_div(m, f.bm) * ceil_div(batch, f.bn);
  return tiles <= kTiles && tiles * f.ksplit * f.bm * f.bn * 4 <= static_cast<int64_t>(kPartBytes);
}

inline int pick(int m, int k, int batch, int cus) {
  int best = 0;
  float least = 0.f;
  for (int i = 0; i < kForms; i++) {
    if (!fits(i, m, batch)) continue;
    const Form &f = kForm[i];
    const int64_t blocks = ceil_div(m, f.bm) * ceil_div(batch, f.bn) * f.ksplit;
    const float steps = static_cast<float>(ceil_div(k, f.k * f.ksplit));
    const float us = f.fixed + steps * (f.step + f.round * static_cast<float>(ceil_div(blocks, cus) - 1)) +
                     f.out * static_cast<float>(m) * static_cast<float>(batch) * 1e-6f;
    if (i == 0 || us < least) {
      best = i;
      least = us;
    }
  }
  return best;
}

}  // namespace rowsform
}  // namespace xe
