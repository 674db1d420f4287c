// paged_attn.hip -- attention of one new token a stream over the keys and
// values in its pages.
#include "attn_dev.h"
#include "paged.h"

namespace xe {
namespace {

constexpr int kT = 256;

// One workgroup a (stream, query head): 256 keys at a time, a key a thread.
template <int HD>
__global__ __launch_bounds__(kT) void paged_attn_kernel(PagedAttn a) {
  __shared__ float q[HD], w[kT], red[kT / 64], acc[kT];
  const int h = blockIdx.x, b = blockIdx.y, t = threadIdx.x;
  const int kvh = h / (a.hq / a.kv.hkv), lane = t & 63, wave = t >> 6;
  const int32_t *row = a.kv.table + static_cast<size_t>(b) * a.kv.max_pages;
  if (t < HD) q[t] = a.q[static_cast<size_t>(b) * a.ldq + h * HD + t];
  int lo, hi;
  paged::key_range(a.lens[b], a.window, a.kv.max_pages << a.kv.page_shift, lo, hi);
  const int mask = (1 << a.kv.page_shift) - 1;
  constexpr int KG = kT / HD;  // keys whose values are added at once
  float m = -INFINITY, l = 0.f, o = 0.f;
  __syncthreads();
  for (int k0 = lo; k0 < hi; k0 += kT) {
    const int key = k0 + t;
    const int page = key < hi ? paged::page_of(row, a.kv.max_pages, a.kv.n_pages, a.kv.page_shift, key) : -1;
    float s = -INFINITY;
    if (page >= 0) {
      const uint16_t *k = a.kv.k + paged::row_at(a.kv.page_stride, a.kv.page_shift, HD, page, kvh, key & mask);
      s = 0.f;
      for (int d = 0; d < HD; d++) s += q[d] * __uint_as_float(static_cast<uint32_t>(k[d]) << 16);
      s *= a.scale * adev::kLog2e;
    }
    float mx = gdev::wave_max(s);
    if (lane == 0) red[wave] = mx;
    __syncthreads();
    const float mn = fmaxf(m, fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3])));
    const float mu = mn == -INFINITY ? 0.f : mn;
    const float p = page >= 0 ? __builtin_amdgcn_exp2f(s - mu) : 0.f, corr = __builtin_amdgcn_exp2f(m - mu);
    m = mn;
    w[t] = p;
    const float ps = gdev::wave_sum(p);
    __syncthreads();
    if (lane == 0) red[wave] = ps;
    __syncthreads();
    l = l * corr + red[0] + red[1] + red[2] + red[3];
    o *= corr;
    for (int i = t / HD; i < kT && k0 + i < hi; i += KG) {
      const int pg = paged::page_of(row, a.kv.max_pages, a.kv.n_pages, a.kv.page_shift, k0 + i);
      if (pg < 0) continue;
      const uint16_t *v = a.kv.v + paged::row_at(a.kv.page_stride, a.kv.page_shift, HD, pg, kvh, (k0 + i) & mask);
      o += w[i] * __uint_as_float(static_cast<uint32_t>(v[t % HD]) << 16);
    }
    __syncthreads();
  }
  acc[t] = o;
  __syncthreads();
  if (t < HD) {
    for (int i = 1; i < KG; i++) o += acc[t + i * HD];
    a.out[static_cast<size_t>(b) * a.ldo + h * HD + t] = l > 0.f ? o / l : (l == 0.f ? 0.f : o);
  }
}

}  // namespace

void launch_paged_attn(const PagedAttn &a, hipStream_t s) {
  auto fn = a.kv.hd == 64 ? paged_attn_kernel<64> : a.kv.hd == 128 ? paged_attn_kernel<128> : paged_attn_kernel<256>;
  hipLaunchKernelGGL(fn, dim3(a.hq, a.kv.batch), dim3(kT), 0, s, a);
  XE_HIP(hipGetLastError());
}

}  // namespace xe
