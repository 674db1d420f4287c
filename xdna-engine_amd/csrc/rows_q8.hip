// rows_q8.hip -- int8 linears whose activations have a scale a row: residual
// addition, norm and quantisation of each row, then an int8 MFMA GEMM with
// bias, activation and residual in its epilogue.
//
// q = round(h / s), s = max|h| / 127 a row: a stream's result does not depend
// on the streams beside it (xe_w8a8_linear has one scale for all rows).
// Statistics and rounding are in fp64, so that a code between two values does
// not depend on the order of a sum: q and s are those of h itself.
#include <type_traits>

#include "attn_dev.h"
#include "paged.h"
#include "rows_form.h"

namespace xe {
namespace {

constexpr unsigned kNoRec = 0x7ffffff0u;  // past every buffer: loads return zeros

constexpr int kXcds = 8;
constexpr size_t kPartBytes = rowsform::kPartBytes;  // partial tiles of K splits
constexpr size_t kCntWords = rowsform::kTiles;       // and their arrival counters
constexpr int kMaxSplit = 4;        // parts of K
constexpr int kStep = 128;          // bytes of K a step
constexpr int kFusedK = rowsform::kFusedK;

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

// Raw buffer over `bytes` bytes: loads past its end give zeros.
__device__ __forceinline__ __amdgpu_buffer_rsrc_t bounded_rsrc(const void *base, unsigned bytes) {
  const uint64_t a = reinterpret_cast<uint64_t>(base);
  const uint64_t lo = static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(static_cast<uint32_t>(a)));
  const uint64_t hi = static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(static_cast<uint32_t>(a >> 32)));
  return __builtin_amdgcn_make_buffer_rsrc(reinterpret_cast<void *>(hi << 32 | lo), static_cast<short>(0),
                                           static_cast<int>(__builtin_amdgcn_readfirstlane(bytes)), 0x00020000);
}

// A double moved by a 32-bit lane move of its halves.
template <typename F>
__device__ __forceinline__ double moved(double v, F &&move) {
  const uint64_t u = __builtin_bit_cast(uint64_t, v);
  const uint32_t lo = move(static_cast<uint32_t>(u)), hi = move(static_cast<uint32_t>(u >> 32));
  return __builtin_bit_cast(double, static_cast<uint64_t>(hi) << 32 | lo);
}
template <int CTRL>
__device__ __forceinline__ double dpp64(double v) {
  return moved(v, [](uint32_t x) { return static_cast<uint32_t>(gdev::dpp_get_i<CTRL>(static_cast<int>(x))); });
}
template <bool HALF>  // the value of the other 32 lanes (HALF) or of the neighbouring 16
__device__ __forceinline__ double other64(double v) {
  return moved(v, [](uint32_t x) {
    const auto r = HALF ? __builtin_amdgcn_permlane32_swap(x, x, false, false) : __builtin_amdgcn_permlane16_swap(x, x, false, false);
    return (threadIdx.x & (HALF ? 32 : 16)) ? r[0] : r[1];
  });
}
// op over all T threads of the workgroup, or over the wave (T = 64), the same in
// each; red: T / 64 doubles of a slot that no wave still reads (T = 64: none).
template <int T, typename Op>
__device__ __forceinline__ double block_all(double v, double *red, Op op) {
  v = op(v, dpp64<gdev::kDppXor1>(v));
  v = op(v, dpp64<gdev::kDppXor2>(v));
  v = op(v, dpp64<gdev::kDppHalfMirror>(v));
  v = op(v, dpp64<gdev::kDppMirror>(v));
  v = op(v, other64<false>(v));
  v = op(v, other64<true>(v));
  if constexpr (T == 64) return v;
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  v = red[0];
#pragma unroll
  for (int w = 1; w < T / 64; w++) v = op(v, red[w]);
  return v;
}
struct Sum64 {
  __device__ double operator()(double a, double b) const { return a + b; }
};
struct Max64 {
  __device__ double operator()(double a, double b) const { return fmax(a, b); }
};

template <bool VEC>
__device__ __forceinline__ f32x4 load4(const float *p) {
  if constexpr (VEC) return *reinterpret_cast<const f32x4 *>(p);
  else return f32x4{p[0], p[1], p[2], p[3]};
}

// Codes lie as the matrix instruction takes them: a block of 1 KB for 64 k of 16
// rows, [kp / 64][groups of 16 rows][4 x 16 k][16 rows][16 k], zeros behind K.  A
// wave loads such an operand as one run of memory (112 B/ns a CU out of L2, 37
// where 16 rows of 64 bytes lie apart); rows behind the last one are whatever is
// there, and so are the results that nobody takes.
__host__ __device__ __forceinline__ int row_groups(int batch) { return (batch + 15) / 16; }
__device__ __forceinline__ size_t code_at(const RowsQ8 &p, int b, int i) {
  return ((static_cast<size_t>(i / 64) * row_groups(p.a.batch) + b / 16) * 64 + i % 64 / 16 * 16 + b % 16) * 16 + i % 16;
}

// h / s is taken as h r with r = 1 / s, within 2^-46 of it for codes up to 127, so
// a half may come out just below one: 2^-44 more than a half lifts it.  The
// quotient of two fp32 values that is no half is 2^-26 or more away from one;
// behind a norm h itself is known to about 2^-44.
constexpr double kHalf = 0.5 + 0x1p-44;

// Row b to codes by T threads, a thread holding elements 4 (tid + T j) .. + 3:
// put(i, four codes) for each four below kp, the scale returned.  `sum` is
// written where `writes`.  red: four slots of T / 64 (T = 64: none).
template <int NV, int T, bool VEC, typename Put>
__device__ __forceinline__ float quant_row(const RowsQ8 &p, int b, bool writes, double *red, Put &&put) {
  const int K = p.k, tid = threadIdx.x % T;
  const size_t at = static_cast<size_t>(b) * K;
  // All loads of the row in flight at once where 4 waves a SIMD leave registers
  // for them (128 each), otherwise the norms' where they are used.
  constexpr bool kEarly = T < 1024;
  f32x4 t[NV], su[NV], pw[NV], g[NV], be[NV];
  auto load = [&](f32x4(&v)[NV], const float *src, auto vec) {
#pragma unroll
    for (int j = 0; j < NV; j++) v[j] = load4<decltype(vec)::value>(src + min(4 * (tid + T * j), K - 4));
  };
  constexpr std::bool_constant<VEC> vec;
  load(t, p.a.x + at, vec);
  if (p.a.add) load(su, p.a.add + at, vec);
  if (p.a.post_w) load(pw, p.a.post_w, vec);
  if (kEarly && p.norm != XE_NORM_NONE) load(g, p.gamma, std::true_type{});
  if (kEarly && p.norm == XE_NORM_LN) load(be, p.beta, std::true_type{});
  if (p.a.post_w) {
    double v = 0.0;
#pragma unroll
    for (int j = 0; j < NV; j++)
#pragma unroll
      for (int c = 0; c < 4; c++)
        if (4 * (tid + T * j) < K) v = __builtin_fma(static_cast<double>(su[j][c]), static_cast<double>(su[j][c]), v);
    const double inv = 1.0 / sqrt(block_all<T>(v, red + 0 * (T / 64), Sum64{}) / K + static_cast<double>(p.a.post_eps));
#pragma unroll
    for (int j = 0; j < NV; j++)
#pragma unroll
      for (int c = 0; c < 4; c++) su[j][c] = static_cast<float>(su[j][c] * inv * (1.0 + pw[j][c]));
  }
  if (p.a.add)
#pragma unroll
    for (int j = 0; j < NV; j++)
#pragma unroll
      for (int c = 0; c < 4; c++) t[j][c] += su[j][c];
#pragma unroll
  for (int j = 0; j < NV; j++) {
    const int i = 4 * (tid + T * j);
    if (p.a.sum && writes && i < K) {
      if constexpr (VEC) *reinterpret_cast<f32x4 *>(p.a.sum + at + i) = t[j];
      else
#pragma unroll
        for (int c = 0; c < 4; c++) p.a.sum[at + i + c] = t[j][c];
    }
    if (i >= K) t[j] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  double h[NV][4];
#pragma unroll
  for (int j = 0; j < NV; j++)
#pragma unroll
    for (int c = 0; c < 4; c++) h[j][c] = t[j][c];
  if (p.norm != XE_NORM_NONE) {
    if (!kEarly) load(g, p.gamma, std::true_type{});
    double v = 0.0;
    if (p.norm == XE_NORM_LN) {
#pragma unroll
      for (int j = 0; j < NV; j++)
#pragma unroll
        for (int c = 0; c < 4; c++) v += h[j][c];
      const double mean = block_all<T>(v, red + 1 * (T / 64), Sum64{}) / K;
      v = 0.0;
#pragma unroll
      for (int j = 0; j < NV; j++)
#pragma unroll
        for (int c = 0; c < 4; c++) h[j][c] = 4 * (tid + T * j) < K ? h[j][c] - mean : 0.0;
    }
#pragma unroll
    for (int j = 0; j < NV; j++)
#pragma unroll
      for (int c = 0; c < 4; c++) v = __builtin_fma(h[j][c], h[j][c], v);
    const double inv = 1.0 / sqrt(block_all<T>(v, red + 2 * (T / 64), Sum64{}) / K + static_cast<double>(p.eps));
    const double one = p.norm == XE_NORM_RMS1P ? 1.0 : 0.0;
#pragma unroll
    for (int j = 0; j < NV; j++)
#pragma unroll
      for (int c = 0; c < 4; c++) h[j][c] = h[j][c] * inv * (one + g[j][c]);
    if (p.norm == XE_NORM_LN) {
      if (!kEarly) load(be, p.beta, std::true_type{});
#pragma unroll
      for (int j = 0; j < NV; j++)
#pragma unroll
        for (int c = 0; c < 4; c++) h[j][c] = 4 * (tid + T * j) < K ? h[j][c] + be[j][c] : 0.0;
    }
  }
  double a = 0.0, bad = 0.0;  // bad: NaN once a value is NaN or infinite
#pragma unroll
  for (int j = 0; j < NV; j++)
#pragma unroll
    for (int c = 0; c < 4; c++) {
      a = fmax(a, fabs(h[j][c]));
      bad = __builtin_fma(h[j][c], 0.0, bad);
    }
  const double amax = block_all<T>(bad == 0.0 ? a : INFINITY, red + 3 * (T / 64), Max64{});
  float s = static_cast<float>(amax / 127.0);
  if (!(s > 0.f)) s = 1.f;
  const bool number = s < INFINITY;  // else NaN or infinity in the row: its scale, and its outputs, become NaN
  const double r = 1.0 / static_cast<double>(s);
#pragma unroll
  for (int j = 0; j < NV; j++) {
    const int i = 4 * (tid + T * j);
    if (i >= p.kp) continue;
    uint32_t q = 0;
#pragma unroll
    for (int c = 0; c < 4; c++) {  // half a unit away from zero, then cut; a scale below fp32's normal range may leave more than 127
      const int code = static_cast<int>(__builtin_fma(h[j][c], r, copysign(kHalf, h[j][c])));
      q |= (static_cast<uint32_t>(min(max(code, -127), 127)) & 0xffu) << (8 * c);
    }
    put(i, number && i < K ? q : 0u);
  }
  return number ? s : NAN;
}

// One workgroup a row, as few threads as hold it in 16 elements each.  Bound by
// the chain of a load and two or three block reductions where rows are few (64 of
// 4096: 3.5 us), by fp64 instructions where they are many (512 of 4096 8.6, 200 of
// 14336 7.3; the rows' bytes 2.2 and 3).  Rounding by a multiply-add and a
// conversion, loads all ahead and h kept took these from 4.9, 11.0 and 9.6.  Half
// the threads with twice the elements: 200 of 14336 1.4 us more; twice the
// threads: 300 of 8192 0.7 more.  K beyond 16384 spills 90 registers.
template <int NV, int T, bool VEC>
__global__ __launch_bounds__(T) void rows_quant_kernel(RowsQ8 p) {
  __shared__ double red[4 * (T / 64)];
  const int b = blockIdx.x;
  const float s = quant_row<NV, T, VEC>(p, b, true, red, [&](int i, uint32_t q) {
    *reinterpret_cast<uint32_t *>(p.codes + code_at(p, b, i)) = q;
  });
  if (threadIdx.x == 0) p.scales[b] = s;
}

__device__ __forceinline__ float gelu_tanh_f(float x) {
  const float u = 0.7978845608028654f * (x + 0.044715f * x * x * x);
  return 0.5f * x * (1.0f + tanhf(u));
}
__device__ __forceinline__ float activate(int act, float z) {
  if (act == XE_ACT_RELU) return z < 0.f ? 0.f : z;
  if (act == XE_ACT_GELU) return 0.5f * z * (1.0f + erff(z * 0.70710678118654752f));
  if (act == XE_ACT_SILU) return z / (1.0f + expf(-z));
  return z;
}

// Outputs r .. r + 3 of activation row b from their sums: what they take is
// loaded early (rows and weight rows past the last one: the last one's).
struct Epi4 {
  float s, ws[4], bi[4], e[4];
  __device__ __forceinline__ void load(const RowsQ8 &p, int b, int r, bool scale) {
    b = min(b, p.a.batch - 1);
    const bool pairs = p.a.act == XE_ACT_GEGLU;
    const int mo = pairs ? p.m / 2 : p.m;
    if (scale) s = p.scales[b];
    if (p.vec) {
      r = min(r, p.m - 4);
      const f32x4 w4 = *reinterpret_cast<const f32x4 *>(p.ws + r);
      f32x4 b4 = {0.f, 0.f, 0.f, 0.f}, e4 = b4;
      if (p.bias) b4 = *reinterpret_cast<const f32x4 *>(p.bias + r);
      if (p.a.res && pairs) {
        const f32x2 e2 = *reinterpret_cast<const f32x2 *>(p.a.res + static_cast<size_t>(b) * mo + r / 2);
        e4[0] = e2[0];
        e4[2] = e2[1];
      } else if (p.a.res) {
        e4 = *reinterpret_cast<const f32x4 *>(p.a.res + static_cast<size_t>(b) * mo + r);
      }
#pragma unroll
      for (int i = 0; i < 4; i++) {
        ws[i] = w4[i];
        bi[i] = b4[i];
        e[i] = e4[i];
      }
      return;
    }
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const int ri = min(r + i, p.m - 1);
      ws[i] = p.ws[ri];
      bi[i] = p.bias ? p.bias[ri] : 0.f;
      e[i] = p.a.res ? p.a.res[static_cast<size_t>(b) * mo + (pairs ? ri / 2 : ri)] : 0.f;
    }
  }
  __device__ __forceinline__ void finish(const RowsQ8 &p, int b, int r, const i32x4 &sum) const {
    const bool pairs = p.a.act == XE_ACT_GEGLU;
    const int mo = pairs ? p.m / 2 : p.m;
    float y[4];
#pragma unroll
    for (int i = 0; i < 4; i++) {
      y[i] = static_cast<float>(sum[i]) * s * ws[i];
      if (p.bias) y[i] += bi[i];
    }
    if (pairs) {
      y[0] = gelu_tanh_f(y[0]) * y[1];
      y[2] = gelu_tanh_f(y[2]) * y[3];
    } else {
#pragma unroll
      for (int i = 0; i < 4; i++) y[i] = activate(p.a.act, y[i]);
    }
    if (p.a.res)
#pragma unroll
      for (int i = 0; i < 4; i++) y[i] += e[i];
    float *d = p.a.y + static_cast<size_t>(b) * mo + (pairs ? r / 2 : r);
    if (p.vec && pairs) {
      *reinterpret_cast<f32x2 *>(d) = f32x2{y[0], y[2]};
    } else if (p.vec) {
      *reinterpret_cast<f32x4 *>(d) = f32x4{y[0], y[1], y[2], y[3]};
    } else {
#pragma unroll
      for (int i = 0; i < 4; i++)
        if (r + i < p.m && !(pairs && (i & 1))) d[pairs ? i / 2 : i] = y[i];
    }
  }
};

// Tiles of WR x 16 weight rows and NJ x 16 activation rows a workgroup, its KS
// waves each over their own part of K (v_mfma_i32_16x16x64_i8: a lane holds 16
// consecutive k of weight row lane % 16 and of activation row lane % 16), U
// steps of 64 in flight.  NV > 0: the workgroup makes the codes itself, into LDS,
// while its first weights load: one row (K <= 1024 NV), or (MANY) a row a wave (K
// <= 256 NV).  Bound by the weights'
// way to the CUs: 64 x 4096 -> 4096 8.4 us for 17 MB of weights (3.5 at a large
// copy's 4.86 TB/s) that two tiles of rows each read; one row 1152 -> 13824 7.4 for
// 16 MB.  The waves' sums meet in LDS.  A CU draws such rows of 64 bytes at 37 B/ns,
// so that few tiles of a long K are bound by that: parts of K (ksplit) go to
// other CUs then and leave their sums in `part`; the last workgroup of a tile to
// arrive adds them, integers, so that their order changes nothing.
template <int WR, int NJ, int KS, int U, int NV, bool MANY>
__global__ __launch_bounds__(64 * KS) void rows_gemm_kernel(RowsQ8 p, int ntile_m, int ntile_b, int ksplit) {
  constexpr int NB = WR * NJ;                     // 16 x 16 blocks
  constexpr bool kFused = NV > 0;
  static_assert(!kFused || (KS == (MANY ? 8 : 4) && NJ == 1), "one row by 256 threads, or a row a wave");
  __shared__ __attribute__((aligned(16))) int part[KS][NB][256];
  __shared__ __attribute__((aligned(16))) int8_t codes[MANY ? 256 * 16 * NV : kFused ? kFusedK : 16];
  __shared__ double red[kFused && !MANY ? 16 : 1];
  __shared__ float made[16];
  __shared__ int flag;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int ln = lane & 15, lg = lane >> 4;
  // The tiles of an XCD lie in a row, those of the same weights next to each
  // other: its L2 reads the weights once.
  const int all = ntile_m * ntile_b * ksplit, each = (all + kXcds - 1) / kXcds;
  const int at = static_cast<int>(blockIdx.x % kXcds) * each + static_cast<int>(blockIdx.x / kXcds);
  if (static_cast<int>(blockIdx.x / kXcds) >= each || at >= all) return;
  const int tb = at % ntile_b, rest = at / ntile_b, kz = rest % ksplit, tm = rest / ksplit;
  const int r0 = tm * 16 * WR, b0 = tb * 16 * NJ;
  const int kp = p.kp;
  const __amdgpu_buffer_rsrc_t rw = bounded_rsrc(p.w, static_cast<unsigned>(p.m) * p.k);
  const int groups = row_groups(p.a.batch);
  const __amdgpu_buffer_rsrc_t ra = bounded_rsrc(p.codes, static_cast<unsigned>(groups) * 16 * kp);
  unsigned wo[WR], xo[NJ];
#pragma unroll
  for (int r = 0; r < WR; r++) wo[r] = r0 + 16 * r + ln < p.m ? static_cast<unsigned>(r0 + 16 * r + ln) * p.k + 16 * lg : kNoRec;
#pragma unroll
  for (int j = 0; j < NJ; j++) xo[j] = tb * NJ + j < groups ? static_cast<unsigned>(tb * NJ + j) * 1024 + 16 * lane : kNoRec;
  const int steps = (p.k + 63) / 64, slot = kz * KS + wave, q = steps / (KS * ksplit), rem = steps % (KS * ksplit);
  const int s0 = q * slot + min(slot, rem), s1 = s0 + q + (slot < rem ? 1 : 0);
  i32x4 w[U][WR], x[U][NJ];
  auto issue = [&](int u, int s) {  // past the last step: zeros
    const bool ok = s < s1;
#pragma unroll
    for (int r = 0; r < WR; r++)
      w[u][r] = __builtin_bit_cast(i32x4, __builtin_amdgcn_raw_buffer_load_b128(rw, ok ? wo[r] : kNoRec, 64 * s, 0));
    if constexpr (!kFused) {
#pragma unroll
      for (int j = 0; j < NJ; j++)
        x[u][j] = __builtin_bit_cast(i32x4, __builtin_amdgcn_raw_buffer_load_b128(ra, ok ? xo[j] : kNoRec, s * groups * 1024, 0));
    }
  };
  i32x4 acc[NB];
#pragma unroll
  for (int i = 0; i < NB; i++) acc[i] = i32x4{0, 0, 0, 0};
#pragma unroll
  for (int u = 0; u < U; u++) issue(u, s0 + u);
  // the epilogue's scales of this lane's first block, in flight too
  const int ob = b0 + 16 * (wave % NJ) + ln, orow = r0 + 16 * (wave / NJ) + 4 * lg;
  Epi4 epi;
  if (wave < NB) epi.load(p, ob, orow, !kFused);
  if constexpr (MANY) {
    const float s = quant_row<NV, 64, true>(p, min(wave, p.a.batch - 1), tm == 0 && wave < p.a.batch, nullptr, [&](int i, uint32_t c) {
      *reinterpret_cast<uint32_t *>(codes + ((i / 64 * 4 + i % 64 / 16) * 16 + wave) * 16 + i % 16) = c;
    });
    if (lane == 0) made[wave] = s;
    __syncthreads();
    epi.s = made[ln];
  } else if constexpr (kFused) {
    epi.s = quant_row<NV, 256, true>(p, 0, at == 0, red, [&](int i, uint32_t c) { *reinterpret_cast<uint32_t *>(codes + i) = c; });
    __syncthreads();
  }
  for (int s = s0; s < s1; s += U) {
#pragma unroll
    for (int u = 0; u < U; u++) {
      if constexpr (MANY) x[u][0] = *reinterpret_cast<const i32x4 *>(codes + min(s + u, kp / 64 - 1) * 1024 + 16 * lane);
      else if constexpr (kFused) x[u][0] = *reinterpret_cast<const i32x4 *>(codes + min(64 * (s + u), kp - 64) + 16 * lg);
#pragma unroll
      for (int r = 0; r < WR; r++)
#pragma unroll
        for (int j = 0; j < NJ; j++)
          acc[r * NJ + j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(w[u][r], x[u][j], acc[r * NJ + j], 0, 0, 0);
      issue(u, s + u + U);
    }
  }
#pragma unroll
  for (int i = 0; i < NB; i++) *reinterpret_cast<i32x4 *>(&part[wave][i][4 * lane]) = acc[i];
  __syncthreads();
  auto waves_sum = [&](int i) {
    i32x4 sum = *reinterpret_cast<const i32x4 *>(&part[0][i][4 * lane]);
#pragma unroll
    for (int k = 1; k < KS; k++) {
      const i32x4 v = *reinterpret_cast<const i32x4 *>(&part[k][i][4 * lane]);
#pragma unroll
      for (int c = 0; c < 4; c++) sum[c] += v[c];
    }
    return sum;
  };
  auto finish = [&](int i, const i32x4 &sum) {
    const int b = b0 + 16 * (i % NJ) + ln, r = r0 + 16 * (i / NJ) + 4 * lg;
    if (i != wave) epi.load(p, b, r, !kFused);
    if (b < p.a.batch && r < p.m) epi.finish(p, b, r, sum);
  };
  if (kFused || ksplit == 1) {
    for (int i = wave; i < NB; i += KS) finish(i, waves_sum(i));
    return;
  }
  const size_t tile = static_cast<size_t>(tm) * ntile_b + tb;
  const __amdgpu_buffer_rsrc_t rp = gdev::coherent_rsrc(reinterpret_cast<const i32x4 *>(p.part) + tile * ksplit * NB * 64);
  for (int i = wave; i < NB; i += KS)
    __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, waves_sum(i)), rp, ((kz * NB + i) * 64 + lane) * 16, 0,
                                           gdev::kCoherentSc1);
  if (!adev::last_to_arrive(p.cnt + tile, ksplit, &flag)) return;
  if (threadIdx.x == 0) __hip_atomic_store(p.cnt + tile, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  for (int i = wave; i < NB; i += KS) {
    i32x4 v[kMaxSplit], sum = {0, 0, 0, 0};
#pragma unroll
    for (int o = 0; o < kMaxSplit; o++)  // past the last one: that one again, not added
      v[o] = __builtin_bit_cast(i32x4, __builtin_amdgcn_raw_buffer_load_b128(rp, ((min(o, ksplit - 1) * NB + i) * 64 + lane) * 16, 0,
                                                                             gdev::kCoherentSc1));
#pragma unroll
    for (int o = 0; o < kMaxSplit; o++)
#pragma unroll
      for (int c = 0; c < 4; c++) sum[c] += o < ksplit ? v[o][c] : 0;
    finish(i, sum);
  }
}

// Outputs of NR activation rows x W C weight rows whose sums lie in LDS, rows
// of `stride`: lane l has weight rows r0 + W (l % C) .. + W - 1 of every (64 /
// C)th activation row, so that a row's outputs leave side by side.  The
// residuals of four or eight rows load together.  ws, bi: of the lane's weight rows.
template <int ACT, int W, int C, int NR>
__device__ __forceinline__ void rows_out(const RowsQ8 &p, const int *sums, int stride, int b0, int bj, int r0, const float *sc,
                                         const float (&ws)[W], const float (&bi)[W]) {
  constexpr int NO = ACT == XE_ACT_GEGLU ? W / 2 : W;  // outputs of a lane
  constexpr int RW = 64 / C, M = W == 4 ? 4 : 8, U = NR / RW < M ? NR / RW : M;  // rows at once
  const int lane = threadIdx.x & 63, c = W * (lane % C), r = r0 + c;
  if (r >= p.m) return;
  const int mo = ACT == XE_ACT_GEGLU ? p.m / 2 : p.m, ro = ACT == XE_ACT_GEGLU ? r / 2 : r;
  typedef float OutV __attribute__((ext_vector_type(NO)));
  typedef int SumV __attribute__((ext_vector_type(W)));
#pragma unroll 1
  for (int i0 = lane / C; i0 < NR; i0 += U * RW) {
    float e[U][NO];
    if (p.a.res) {
#pragma unroll
      for (int u = 0; u < U; u++) {
        const OutV v = *reinterpret_cast<const OutV *>(p.a.res + static_cast<size_t>(min(b0 + bj + i0 + u * RW, p.a.batch - 1)) * mo + ro);
#pragma unroll
        for (int i = 0; i < NO; i++) e[u][i] = v[i];
      }
#pragma unroll
      for (int u = 0; u < U; u++)
#pragma unroll
        for (int i = 0; i < NO; i++) asm volatile("" : "+v"(e[u][i]));  // none is moved to where it is used
    }
#pragma unroll
    for (int u = 0; u < U; u++) {
      const int row = i0 + u * RW, b = b0 + bj + row;
      if (b >= p.a.batch) continue;
      const SumV v = *reinterpret_cast<const SumV *>(sums + row * stride + c);
      const float s = sc[bj + row];
      float z[W];
#pragma unroll
      for (int i = 0; i < W; i++) {
        z[i] = static_cast<float>(v[i]) * s * ws[i];
        if (p.bias) z[i] += bi[i];
      }
      OutV y;
#pragma unroll
      for (int i = 0; i < NO; i++) {
        if constexpr (ACT == XE_ACT_GEGLU) y[i] = gelu_tanh_f(z[2 * i]) * z[2 * i + 1];
        else y[i] = activate(ACT, z[i]);
      }
      if (p.a.res)
#pragma unroll
        for (int i = 0; i < NO; i++) y[i] += e[u][i];
      *reinterpret_cast<OutV *>(p.a.y + static_cast<size_t>(b) * mo + ro) = y;
    }
  }
}
// The same for all activations: four weight rows a lane where results go out
// that wide, else one output a lane, up to 64 side by side (512 x 4096 -> 14338 63
// us with four values a lane one by one, 54 so; 64 x 4096 -> 4098 16.7 and 14.9).
template <int MW, int NR>
__device__ __forceinline__ void rows_out_any(const RowsQ8 &p, const int *sums, int stride, int b0, int bj, int r0, const float *sc,
                                             const float (&ws)[4], const float (&bi)[4]) {
  if (p.vec) {
    switch (p.a.act) {
      case XE_ACT_RELU: return rows_out<XE_ACT_RELU, 4, MW / 4, NR>(p, sums, stride, b0, bj, r0, sc, ws, bi);
      case XE_ACT_GELU: return rows_out<XE_ACT_GELU, 4, MW / 4, NR>(p, sums, stride, b0, bj, r0, sc, ws, bi);
      case XE_ACT_SILU: return rows_out<XE_ACT_SILU, 4, MW / 4, NR>(p, sums, stride, b0, bj, r0, sc, ws, bi);
      case XE_ACT_GEGLU: return rows_out<XE_ACT_GEGLU, 4, MW / 4, NR>(p, sums, stride, b0, bj, r0, sc, ws, bi);
      default: return rows_out<XE_ACT_NONE, 4, MW / 4, NR>(p, sums, stride, b0, bj, r0, sc, ws, bi);
    }
  }
  const float w1[1] = {ws[0]}, b1[1] = {bi[0]}, w2[2] = {ws[0], ws[1]}, b2[2] = {bi[0], bi[1]};
  switch (p.a.act) {
    case XE_ACT_RELU: return rows_out<XE_ACT_RELU, 1, MW, NR>(p, sums, stride, b0, bj, r0, sc, w1, b1);
    case XE_ACT_GELU: return rows_out<XE_ACT_GELU, 1, MW, NR>(p, sums, stride, b0, bj, r0, sc, w1, b1);
    case XE_ACT_SILU: return rows_out<XE_ACT_SILU, 1, MW, NR>(p, sums, stride, b0, bj, r0, sc, w1, b1);
    case XE_ACT_GEGLU: return rows_out<XE_ACT_GEGLU, 2, MW / 2, NR>(p, sums, stride, b0, bj, r0, sc, w2, b2);
    default: return rows_out<XE_ACT_NONE, 1, MW, NR>(p, sums, stride, b0, bj, r0, sc, w1, b1);
  }
}

// Tiles of BM weight rows x BN activation rows a workgroup, WV waves of 2 BM / WV
// x BN / 2; K in steps of 128 bytes through two LDS buffers, the loads of two
// more steps in registers.  Rows lie 128 bytes apart in LDS, their 16-byte
// chunks permuted by the row, so that 16 rows read together cover all banks.
// Parts of K as above.  Bound by the matrix instructions and the LDS reads that
// feed them: 512 x 4096 -> 14336 in 256 x 128 tiles 41.0 us, 1470 TOP/s on 224 of
// 256 CUs with its start and 29 MB of results (such instructions with such reads
// alone 2650 on all CUs, without reads 3500; a large product of the library 1781).
// A third LDS buffer, so that reads never follow a barrier: 52.9 us for 52.3 in the
// whole call.  Smaller tiles by what the CUs load: 200 x 14336 -> 4096 in 64 x 64
// tiles and two parts of K 29.0 us for 470 MB of operands out of L2, 16 TB/s (runs
// of 128 bytes reach 17 to 20).
// Eight waves instead of four, 128 x 64 tiles, 512 x 4096 -> 4096: 28.6 -> 27.3.
template <int BM, int BN, int WV>
__global__ __launch_bounds__(64 * WV, 2) void rows_tile_kernel(RowsQ8 p, int ntile_m, int ntile_b, int ksplit) {
  constexpr int T = 64 * WV, MW = BM / (WV / 2), NW = BN / 2;  // a wave's rows of weights, of activations
  constexpr int NA = BM * 8 / T, NX = BN * 8 / T;              // 16-byte chunks a thread loads of each operand
  constexpr int FM = MW / 16, FN = NW / 16;                    // 16 x 16 blocks of a wave
  __shared__ __attribute__((aligned(16))) uint8_t lds[2][(BM + BN) * kStep];
  __shared__ float sc[BN];
  __shared__ int flag;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int ln = lane & 15, lg = lane >> 4, wm = wave >> 1, wn = wave & 1;
  const int all = ntile_m * ntile_b * ksplit, each = (all + kXcds - 1) / kXcds;
  const int at = static_cast<int>(blockIdx.x % kXcds) * each + static_cast<int>(blockIdx.x / kXcds);
  if (static_cast<int>(blockIdx.x / kXcds) >= each || at >= all) return;
  const int tb = at % ntile_b, rest = at / ntile_b, z = rest % ksplit, tm = rest / ksplit;
  const int m0 = tm * BM, b0 = tb * BN;
  const __amdgpu_buffer_rsrc_t rw = bounded_rsrc(p.w, static_cast<unsigned>(p.m) * p.k);
  const int groups = row_groups(p.a.batch);
  const __amdgpu_buffer_rsrc_t ra = bounded_rsrc(p.codes, static_cast<unsigned>(groups) * 16 * p.kp);
  const int steps = p.kp / kStep, q = steps / ksplit, rem = steps % ksplit;
  const int s0 = q * z + min(z, rem), ns = q + (z < rem ? 1 : 0);
  // thread t takes chunk t % 8 of weight rows t / 8 + T / 8 j; wave w the blocks w + WV j
  // of the activations, 64 k of the first 16 rows, of the second, ..
  const int xc = tid & 7, xr = tid >> 3;
  unsigned wo[NA], xo[NX];
#pragma unroll
  for (int j = 0; j < NA; j++) wo[j] = m0 + xr + T / 8 * j < p.m ? static_cast<unsigned>(m0 + xr + T / 8 * j) * p.k + 16 * xc : kNoRec;
#pragma unroll
  for (int j = 0; j < NX; j++) {
    const int h = (wave + WV * j) / (BN / 16), g = (wave + WV * j) % (BN / 16);
    xo[j] = b0 / 16 + g < groups ? static_cast<unsigned>(h * groups + b0 / 16 + g) * 1024 + 16 * lane : kNoRec;
  }
  struct Stage {
    i32x4 w[NA], x[NX];
  } st[2];
  auto issue = [&](int i, Stage &g) {  // past the last step: zeros
    const int s = s0 + i;
    const bool ok = i < ns;
#pragma unroll
    for (int j = 0; j < NA; j++)
      g.w[j] = __builtin_bit_cast(i32x4, __builtin_amdgcn_raw_buffer_load_b128(rw, ok ? wo[j] : kNoRec, s * kStep, 0));
#pragma unroll
    for (int j = 0; j < NX; j++)
      g.x[j] = __builtin_bit_cast(i32x4, __builtin_amdgcn_raw_buffer_load_b128(ra, ok ? xo[j] : kNoRec, s * 2 * groups * 1024, 0));
  };
  const int put_at = xr * kStep + ((xc ^ (xr & 7)) << 4);
  auto put = [&](int buf, const Stage &g) {
#pragma unroll
    for (int j = 0; j < NA; j++) *reinterpret_cast<i32x4 *>(&lds[buf][put_at + T / 8 * j * kStep]) = g.w[j];
#pragma unroll
    for (int j = 0; j < NX; j++) {
      const int h = (wave + WV * j) / (BN / 16), rg = (wave + WV * j) % (BN / 16);
      *reinterpret_cast<i32x4 *>(&lds[buf][(BM + 16 * rg + ln) * kStep + (((4 * h + lg) ^ (ln & 7)) << 4)]) = g.x[j];
    }
  };
  const int wbase = (wm * MW + ln) * kStep, xbase = BM * kStep + (wn * NW + ln) * kStep;
  i32x4 acc[FM][FN];
#pragma unroll
  for (int i = 0; i < FM; i++)
#pragma unroll
    for (int j = 0; j < FN; j++) acc[i][j] = i32x4{0, 0, 0, 0};
  // A step's LDS reads, MFMAs, LDS writes of the next step and loads of the one
  // after the next but one, spread over each other.
  auto step = [&](int buf, int next) {
    constexpr int R = FM + FN, M = FM * FN / R, P = NA + NX;
    i32x4 w[2][FM], x[2][FN];
#pragma unroll
    for (int h = 0; h < 2; h++) {
      const int c = ((4 * h + lg) ^ (ln & 7)) << 4;
#pragma unroll
      for (int i = 0; i < FM; i++) w[h][i] = *reinterpret_cast<const i32x4 *>(&lds[buf][wbase + 16 * i * kStep + c]);
#pragma unroll
      for (int j = 0; j < FN; j++) x[h][j] = *reinterpret_cast<const i32x4 *>(&lds[buf][xbase + 16 * j * kStep + c]);
    }
    put(buf ^ 1, st[buf ^ 1]);
    issue(next, st[buf ^ 1]);
#pragma unroll
    for (int h = 0; h < 2; h++)
#pragma unroll
      for (int i = 0; i < FM; i++)
#pragma unroll
        for (int j = 0; j < FN; j++) acc[i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(w[h][i], x[h][j], acc[i][j], 0, 0, 0);
    __builtin_amdgcn_sched_group_barrier(0x100, R, 0);
#pragma unroll
    for (int i = 0; i < R; i++) {
      __builtin_amdgcn_sched_group_barrier(0x8, M, 0);
      __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
    }
#pragma unroll
    for (int i = 0; i < P; i++) {
      __builtin_amdgcn_sched_group_barrier(0x8, FM * FN / P, 0);
      __builtin_amdgcn_sched_group_barrier(0x200, 1, 0);
      __builtin_amdgcn_sched_group_barrier(0x20, 1, 0);
    }
    __syncthreads();
  };
  issue(0, st[0]);
  issue(1, st[1]);
  // the epilogue's scales: of the tile's activation rows, of a lane's weight rows
  for (int i = tid; i < BN; i += T) sc[i] = b0 + i < p.a.batch ? p.scales[b0 + i] : 0.f;
  float ws4[4], bi4[4];
  {
    const int each = p.vec ? 4 : p.a.act == XE_ACT_GEGLU ? 2 : 1;  // weight rows of a lane in rows_out
    const int r = m0 + wm * MW + each * (lane % (MW / each));
    if (each == 4) {
      const int r4 = min(r, p.m - 4);
      const f32x4 w4 = *reinterpret_cast<const f32x4 *>(p.ws + r4);
      f32x4 b4 = {0.f, 0.f, 0.f, 0.f};
      if (p.bias) b4 = *reinterpret_cast<const f32x4 *>(p.bias + r4);
#pragma unroll
      for (int i = 0; i < 4; i++) {
        ws4[i] = w4[i];
        bi4[i] = b4[i];
      }
    } else {
#pragma unroll
      for (int i = 0; i < 4; i++) {
        const int ri = min(r + min(i, each - 1), p.m - 1);
        ws4[i] = p.ws[ri];
        bi4[i] = p.bias ? p.bias[ri] : 0.f;
      }
    }
  }
  put(0, st[0]);
  issue(2, st[0]);
  __syncthreads();
  int i = 0;
  for (; i + 2 <= ns; i += 2) {
    step(0, i + 3);
    step(1, i + 4);
  }
  if (i < ns) step(0, i + 3);
  if (ksplit > 1) {
    constexpr int W4 = BM * BN / 4;  // i32x4 of a tile
    const size_t tile = static_cast<size_t>(tm) * ntile_b + tb;
    const __amdgpu_buffer_rsrc_t rp = gdev::coherent_rsrc(reinterpret_cast<const i32x4 *>(p.part) + tile * ksplit * W4);
#pragma unroll
    for (int i = 0; i < FM; i++)
#pragma unroll
      for (int j = 0; j < FN; j++)
        __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, acc[i][j]), rp,
                                               static_cast<int>((z * W4 + (i * FN + j) * T + tid) * 16), 0, gdev::kCoherentSc1);
    if (!adev::last_to_arrive(p.cnt + tile, ksplit, &flag)) return;
    if (tid == 0) __hip_atomic_store(p.cnt + tile, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    for (int o = 0; o < ksplit; o++) {
      if (o == z) continue;
#pragma unroll
      for (int i = 0; i < FM; i++)
#pragma unroll
        for (int j = 0; j < FN; j++) {
          const i32x4 v = __builtin_bit_cast(i32x4, __builtin_amdgcn_raw_buffer_load_b128(
              rp, static_cast<int>((o * W4 + (i * FN + j) * T + tid) * 16), 0, gdev::kCoherentSc1));
#pragma unroll
          for (int e = 0; e < 4; e++) acc[i][j][e] += v[e];
        }
    }
  }
  // Sums turn through the wave's part of LDS, so that a row's outputs go out
  // side by side: a lane always has the same four weight rows.
  constexpr int RS = MW + 4, JH = FN > 1 ? 2 : 1;  // 16 JH activation rows at a time
  static_assert(WV * 16 * JH * RS * 4 <= sizeof(lds), "the waves' rows fit the operand buffers");
  int *const out = reinterpret_cast<int *>(&lds[0][0]) + wave * 16 * JH * RS;
#pragma unroll
  for (int j0 = 0; j0 < FN; j0 += JH) {
#pragma unroll
    for (int j = 0; j < JH; j++)
#pragma unroll
      for (int i = 0; i < FM; i++) *reinterpret_cast<i32x4 *>(out + (16 * j + ln) * RS + 16 * i + 4 * lg) = acc[i][j0 + j];
    __builtin_amdgcn_wave_barrier();
    const int bj = wn * NW + 16 * j0, rj = m0 + wm * MW;
    rows_out_any<MW, 16 * JH>(p, out, RS, b0, bj, rj, sc, ws4, bi4);
    __builtin_amdgcn_wave_barrier();
  }
}

// Parts of K leave tiles of bm x bn sums in the workspace.
void check_tiles(int tm, int tb, int ksplit, int bm, int bn) {
  const int64_t tiles = static_cast<int64_t>(tm) * tb;
  XE_REQUIRE(tiles * ksplit <= (1 << 22), "rows gemm: too many tiles for one launch");
  XE_REQUIRE(ksplit == 1 || (ksplit <= kMaxSplit && tiles <= static_cast<int64_t>(kCntWords) &&
                             tiles * ksplit * bm * bn * 4 <= static_cast<int64_t>(kPartBytes)),
             "rows gemm: partial tiles beyond the workspace");
}

template <int WR, int NJ, int KS, int U, int NV = 0, bool MANY = false>
void launch_gemm(const RowsQ8 &r, int ksplit, hipStream_t s) {
  const int tm = (r.m + 16 * WR - 1) / (16 * WR), tb = (r.a.batch + 16 * NJ - 1) / (16 * NJ);
  check_tiles(tm, tb, ksplit, 16 * WR, 16 * NJ);
  const int blocks = (tm * tb * ksplit + kXcds - 1) / kXcds * kXcds;
  hipLaunchKernelGGL((rows_gemm_kernel<WR, NJ, KS, U, NV, MANY>), dim3(blocks), dim3(64 * KS), 0, s, r, tm, tb, ksplit);
  XE_HIP(hipGetLastError());
}

template <int BM, int BN, int WV>
void launch_tile(const RowsQ8 &r, int ksplit, hipStream_t s) {
  const int tm = (r.m + BM - 1) / BM, tb = (r.a.batch + BN - 1) / BN;
  check_tiles(tm, tb, ksplit, BM, BN);
  const int blocks = (tm * tb * ksplit + kXcds - 1) / kXcds * kXcds;
  hipLaunchKernelGGL((rows_tile_kernel<BM, BN, WV>), dim3(blocks), dim3(64 * WV), 0, s, r, tm, tb, ksplit);
  XE_HIP(hipGetLastError());
}

// Whether what one workgroup writes may be what another still reads, were rows
// quantised and products finished in one launch.
bool shares(const RowsQ8 &r, int outs) {
  const size_t in = static_cast<size_t>(r.a.batch) * r.k * 4, out = static_cast<size_t>(r.a.batch) * outs * 4;
  auto meet = [](const float *a, size_t n, const float *b, size_t m) {
    const uintptr_t x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(b);
    return a && b && x < y + m && y < x + n;
  };
  return meet(r.a.sum, in, r.a.x, in) || meet(r.a.sum, in, r.a.add, in) || meet(r.a.sum, in, r.a.res, out) || meet(r.a.sum, in, r.a.y, out) ||
         meet(r.a.y, out, r.a.x, in) || meet(r.a.y, out, r.a.add, in);
}

template <bool VEC>
void launch_quant(const RowsQ8 &r, hipStream_t s) {
  const dim3 rows(r.a.batch);
  if (r.k <= 1024) hipLaunchKernelGGL((rows_quant_kernel<1, 256, VEC>), rows, dim3(256), 0, s, r);
  else if (r.k <= 2048) hipLaunchKernelGGL((rows_quant_kernel<2, 256, VEC>), rows, dim3(256), 0, s, r);
  else if (r.k <= 4096) hipLaunchKernelGGL((rows_quant_kernel<4, 256, VEC>), rows, dim3(256), 0, s, r);
  else if (r.k <= 8192) hipLaunchKernelGGL((rows_quant_kernel<4, 512, VEC>), rows, dim3(512), 0, s, r);
  else if (r.k <= 16384) hipLaunchKernelGGL((rows_quant_kernel<4, 1024, VEC>), rows, dim3(1024), 0, s, r);
  else hipLaunchKernelGGL((rows_quant_kernel<8, 1024, VEC>), rows, dim3(1024), 0, s, r);
  XE_HIP(hipGetLastError());
}

}  // namespace

size_t rows_q8_ws_bytes() { return 2048 + kCntWords * 4 + kPartBytes; }

size_t rows_q8_codes_bytes(int batch, int k) { return static_cast<size_t>(row_groups(batch)) * 16 * ((k + kStep - 1) / kStep * kStep); }

int launch_rows_q8(const RowsQ8 &L, hipStream_t s) {
  RowsQ8 r = L;
  r.kp = (r.k + kStep - 1) / kStep * kStep;
  const int outs = r.a.act == XE_ACT_GEGLU ? r.m / 2 : r.m;
  // whether results of four weight rows go out at once
  const uintptr_t rows_at = reinterpret_cast<uintptr_t>(r.a.y) | reinterpret_cast<uintptr_t>(r.a.res) | static_cast<uintptr_t>(outs) * 4;
  const uintptr_t weights_at = reinterpret_cast<uintptr_t>(r.ws) | reinterpret_cast<uintptr_t>(r.bias);
  r.vec = ((rows_at & (r.a.act == XE_ACT_GEGLU ? 7 : 15)) | (weights_at & 15)) == 0;
  const bool in16 = ((reinterpret_cast<uintptr_t>(r.a.x) | reinterpret_cast<uintptr_t>(r.a.add) | reinterpret_cast<uintptr_t>(r.a.sum) |
                      reinterpret_cast<uintptr_t>(r.a.post_w)) & 15) == 0;
  const rowsform::Way way = in16 && !shares(r, outs) ? rowsform::way(r.m, r.k, r.a.batch, gdev::cu_count()) : rowsform::kTwoLaunches;
  if (way == rowsform::kOneRow || way == rowsform::kOneRowWide) {
    const bool wide = way == rowsform::kOneRowWide;
    if (r.k <= 1024) wide ? launch_gemm<2, 1, 4, 4, 1>(r, 1, s) : launch_gemm<1, 1, 4, 8, 1>(r, 1, s);
    else if (r.k <= 2048) wide ? launch_gemm<2, 1, 4, 4, 2>(r, 1, s) : launch_gemm<1, 1, 4, 8, 2>(r, 1, s);
    else wide ? launch_gemm<2, 1, 4, 4, 4>(r, 1, s) : launch_gemm<1, 1, 4, 8, 4>(r, 1, s);
    return 1;
  }
  if (way == rowsform::kWaveRows) {
    if (r.k <= 768) launch_gemm<1, 1, 8, 2, 3, true>(r, 1, s);
    else launch_gemm<1, 1, 8, 3, 5, true>(r, 1, s);
    return 1;
  }
  if (in16) launch_quant<true>(r, s);
  else launch_quant<false>(r, s);
  switch (rowsform::pick(r.m, r.k, r.a.batch, gdev::cu_count())) {
    case 0: launch_gemm<1, 1, 4, 8>(r, 1, s); break;
    case 1: launch_gemm<1, 2, 4, 4>(r, 1, s); break;
    case 2: launch_gemm<2, 2, 4, 4>(r, 1, s); break;
    case 3: launch_tile<64, 64, 4>(r, 1, s); break;
    case 4: launch_tile<64, 64, 4>(r, 2, s); break;
    case 5: launch_tile<64, 64, 4>(r, 4, s); break;
    case 6: launch_tile<128, 64, 8>(r, 1, s); break;
    case 7: launch_tile<128, 128, 8>(r, 1, s); break;
    case 8: launch_tile<256, 128, 8>(r, 1, s); break;
    case 9: launch_gemm<1, 1, 4, 8>(r, 4, s); break;
    default: launch_gemm<1, 2, 4, 4>(r, 4, s); break;
  }
  return 2;
}

}  // namespace xe
