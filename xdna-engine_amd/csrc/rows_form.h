// rows_form.h -- which form of the int8 rows' product a shape takes.
#pragma once

#include <cstddef>
#include <cstdint>

namespace xe {
namespace rowsform {

constexpr size_t kPartBytes = size_t(32) << 20;  // workspace of partial tiles
constexpr int kTiles = 1024;                     // tiles that have an arrival counter

// The forms and the time, in us, that each is estimated to take:
//   fixed + steps (step + round (rounds - 1)) + out m batch / 10^6
// with `steps` of K a workgroup and `rounds` of workgroups a CU.  The first
// three have four waves that share K, 64 a step; the others take 128 a step and
// split K, if at all, over workgroups.  Fitted to 288 shapes (m 768 to 14336, K
// 768 to 14336, 8 to 512 rows), to 5 % a form.  The form of the least estimate is
// 0.4 % slower than the fastest of all on average, 12 % at most.  Measured us of
// the forms in the order of the table (-: its partial tiles do not fit):
//   m x K        rows
//   4096 x 4096    16    6.2  6.7  8.9   12   10   11   14   19   28
//   4096 x 4096    64     14  9.6  9.0   12   11   12   15   20   33
//   4096 x 14336   64     37   23   20   30   21   18   38   53   84
//   4096 x 14336  200    109   71   68   32   29   32   38   52   83
//   14336 x 4096  200    128   81   70   31   34    -   26   23   35
//   14336 x 4096  512    306  182  155   59    -    -   54   50   45
struct Form {
  int bm, bn, ksplit, kstep;
  float fixed, step, round, out;
};
constexpr int kForms = 9;
constexpr int kInWaves = 3;  // forms whose waves share K
constexpr Form kForm[kForms] = {
    {16, 16, 4, 64, 2.69f, 0.154f, 0.131f, 11.4f},   {16, 32, 4, 64, 2.77f, 0.184f, 0.172f, 4.03f},
    {32, 32, 4, 64, 3.07f, 0.302f, 0.286f, 2.92f},   {64, 64, 1, 128, 3.62f, 0.244f, 0.162f, 1.34f},
    {64, 64, 2, 128, 5.44f, 0.256f, 0.163f, 2.49f},  {64, 64, 4, 128, 6.83f, 0.292f, 0.183f, 3.87f},
    {128, 64, 1, 128, 3.83f, 0.309f, 0.263f, 1.39f}, {128, 128, 1, 128, 4.41f, 0.434f, 0.558f, 1.43f},
    {256, 128, 1, 128, 6.85f, 0.682f, 0.682f, 2.12f}};

inline int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

// Whether the partial tiles of form i have room in the workspace.
inline bool fits(int i, int m, int batch) {
  const Form &f = kForm[i];
  if (i < kInWaves || f.ksplit == 1) return true;
  const int64_t tiles = ceil_div(m, f.bm) * ceil_div(batch, f.bn);
  return tiles <= kTiles && tiles * f.ksplit * f.bm * f.bn * 4 <= static_cast<int64_t>(kPartBytes);
}

inline int pick(int m, int k, int batch, int cus) {
  int best = 0;
  float least = 0.f;
  for (int i = 0; i < kForms; i++) {
    if (!fits(i, m, batch)) continue;
    const Form &f = kForm[i];
    const int64_t blocks = ceil_div(m, f.bm) * ceil_div(batch, f.bn) * (i < kInWaves ? 1 : f.ksplit);
    const float steps = static_cast<float>(ceil_div(k, f.kstep * f.ksplit));
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
