// rows_q8.hip -- int8 linears whose activations have a scale a row: residual
// addition, norm and quantisation of each row, then an int8 MFMA GEMM with
// bias, activation and residual in its epilogue.
//
// q = round(h / s), s = max|h| / 127 a row: a stream's result does not depend
// on the streams beside it (xe_w8a8_linear has one scale for all rows).
// Statistics and rounding are in fp64, so that a code between two values does
// not depend on the order of a sum: q and s are those of h itself.
#include "gemv_dev.h"
#include "paged.h"

namespace xe {
namespace {

constexpr int kT = 256;
constexpr int kNoRec = 0x7ffffff0;  // past every buffer: loads return zeros

typedef int i32x4 __attribute__((ext_vector_type(4)));

__device__ __forceinline__ double wave_sum64(double v) {
#pragma unroll
  for (int off = 32; off >= 1; off >>= 1) v += __shfl_xor(v, off, 64);
  return v;
}
__device__ __forceinline__ double wave_max64(double v) {
#pragma unroll
  for (int off = 32; off >= 1; off >>= 1) v = fmax(v, __shfl_xor(v, off, 64));
  return v;
}

template <typename F>
__device__ __forceinline__ double block_reduce(double v, double *red, F op) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  __syncthreads();
  if (lane == 0) red[wave] = v;
  __syncthreads();
  v = red[0];
  for (int w = 1; w < static_cast<int>(blockDim.x >> 6); w++) v = op(v, red[w]);
  return v;
}

// One workgroup a row; a thread holds elements threadIdx.x + T j.
template <int NE, int T>
__global__ __launch_bounds__(T) void rows_quant_kernel(RowsQ8 p) {
  __shared__ double red[T / 64];
  const int b = blockIdx.x, K = p.k;
  const float *x = p.a.x + static_cast<size_t>(b) * K;
  const float *add = p.a.add ? p.a.add + static_cast<size_t>(b) * K : nullptr;
  auto sum = [](double u, double v) { return u + v; };
  float t[NE], su[NE];
#pragma unroll
  for (int j = 0; j < NE; j++) {
    const int i = threadIdx.x + j * T;
    t[j] = i < K ? x[i] : 0.f;
    su[j] = add && i < K ? add[i] : 0.f;
  }
  if (p.a.post_w) {
    double s = 0.0;
#pragma unroll
    for (int j = 0; j < NE; j++) s += static_cast<double>(su[j]) * su[j];
    const double inv = 1.0 / sqrt(block_reduce(wave_sum64(s), red, sum) / K + static_cast<double>(p.a.post_eps));
#pragma unroll
    for (int j = 0; j < NE; j++) {
      const int i = threadIdx.x + j * T;
      if (i < K) su[j] = static_cast<float>(su[j] * inv * (1.0 + p.a.post_w[i]));
    }
  }
  double h[NE];
#pragma unroll
  for (int j = 0; j < NE; j++) {
    const int i = threadIdx.x + j * T;
    if (add) t[j] += su[j];
    if (p.a.sum && i < K) p.a.sum[static_cast<size_t>(b) * K + i] = t[j];
    h[j] = t[j];
  }
  if (p.norm != XE_NORM_NONE) {
    double mean = 0.0;
    if (p.norm == XE_NORM_LN) {
      double s = 0.0;
#pragma unroll
      for (int j = 0; j < NE; j++) s += h[j];
      mean = block_reduce(wave_sum64(s), red, sum) / K;
    }
    double s = 0.0;
#pragma unroll
    for (int j = 0; j < NE; j++) {
      const int i = threadIdx.x + j * T;
      h[j] = i < K ? h[j] - mean : 0.0;
      s += h[j] * h[j];
    }
    const double inv = 1.0 / sqrt(block_reduce(wave_sum64(s), red, sum) / K + static_cast<double>(p.eps));
#pragma unroll
    for (int j = 0; j < NE; j++) {
      const int i = threadIdx.x + j * T;
      if (i >= K) continue;
      h[j] = h[j] * inv * ((p.norm == XE_NORM_RMS1P ? 1.0 : 0.0) + p.gamma[i]);
      if (p.norm == XE_NORM_LN) h[j] += p.beta[i];
    }
  }
  // NaN and infinity: the row's scale becomes NaN, and with it its outputs
  double a = 0.0;
  bool bad = false;
#pragma unroll
  for (int j = 0; j < NE; j++) {
    a = fmax(a, fabs(h[j]));
    bad |= !(fabs(h[j]) <= 1.7976931348623157e308);
  }
  a = bad ? INFINITY : a;
  const double amax = block_reduce(wave_max64(a), red, [](double u, double v) { return fmax(u, v); });
  const float scale = amax > 0.0 ? static_cast<float>(amax / 127.0) : 1.0f;
  if (threadIdx.x == 0) p.scales[b] = scale < INFINITY ? scale : NAN;
  const double r = 1.0 / static_cast<double>(scale);
#pragma unroll
  for (int j = 0; j < NE; j++) {
    const int i = threadIdx.x + j * T;
    if (i >= K) continue;
    const double v = fmin(fmax(round(h[j] * r), -127.0), 127.0);
    p.codes[static_cast<size_t>(b) * K + i] = scale < INFINITY ? static_cast<int8_t>(static_cast<int>(v)) : static_cast<int8_t>(0);
  }
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

// Four waves of 16 weight rows, 16 activation rows a workgroup.
__global__ __launch_bounds__(kT) void rows_gemm_kernel(RowsQ8 p) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int r0 = blockIdx.x * 64 + wave * 16, b0 = blockIdx.y * 16;
  const __amdgpu_buffer_rsrc_t rw = gdev::coherent_rsrc(p.w);
  const __amdgpu_buffer_rsrc_t ra = gdev::coherent_rsrc(p.codes);
  const int row = r0 + (lane & 15), b = b0 + (lane & 15), kl = 16 * (lane >> 4);
  i32x4 acc = {0, 0, 0, 0};
  for (int k0 = 0; k0 < p.k; k0 += 64) {
    const bool ok = k0 + kl < p.k;
    const i32x4 wa = __builtin_bit_cast(i32x4, __builtin_amdgcn_raw_buffer_load_b128(rw, row < p.m && ok ? row * p.k + k0 + kl : kNoRec, 0, 0));
    const i32x4 xa = __builtin_bit_cast(i32x4, __builtin_amdgcn_raw_buffer_load_b128(ra, b < p.a.batch && ok ? b * p.k + k0 + kl : kNoRec, 0, 0));
    acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(wa, xa, acc, 0, 0, 0);
  }
  if (b >= p.a.batch) return;
  const float s = p.scales[b];
  float z[4];
#pragma unroll
  for (int i = 0; i < 4; i++) {
    const int r = min(r0 + 4 * (lane >> 4) + i, p.m - 1);
    z[i] = static_cast<float>(acc[i]) * s * p.ws[r];
    if (p.bias) z[i] += p.bias[r];
  }
  const bool pairs = p.a.act == XE_ACT_GEGLU;
  const int mo = pairs ? p.m / 2 : p.m;
#pragma unroll
  for (int i = 0; i < 4; i++) {
    if (pairs && (i & 1)) continue;
    const int r = r0 + 4 * (lane >> 4) + i;
    if (r >= p.m) continue;
    float y = pairs ? gelu_tanh_f(z[i]) * z[i + 1 < 4 ? i + 1 : 3] : activate(p.a.act, z[i]);
    const size_t o = static_cast<size_t>(b) * mo + (pairs ? r / 2 : r);
    if (p.a.res) y += p.a.res[o];
    p.a.y[o] = y;
  }
}

}  // namespace

void launch_rows_q8(const RowsQ8 &r, hipStream_t s) {
  const dim3 rows(r.a.batch);
  if (r.k <= 2048) hipLaunchKernelGGL((rows_quant_kernel<8, 256>), rows, dim3(256), 0, s, r);
  else if (r.k <= 8192) hipLaunchKernelGGL((rows_quant_kernel<16, 512>), rows, dim3(512), 0, s, r);
  else hipLaunchKernelGGL((rows_quant_kernel<32, 1024>), rows, dim3(1024), 0, s, r);
  XE_HIP(hipGetLastError());
  hipLaunchKernelGGL(rows_gemm_kernel, dim3((r.m + 63) / 64, (r.a.batch + 15) / 16), dim3(kT), 0, s, r);
  XE_HIP(hipGetLastError());
}

}  // namespace xe
