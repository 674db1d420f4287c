// paged_append.hip -- new tokens' keys and values into the pages of their
// streams, the per-head RMSNorm (1 + w) and the rotation by position applied
// on the way, their queries too.
//
// Bound by the rows' bytes (4 a value in; keys and values 2, queries 4 out),
// and for a few rows by one launch and its chain of loads: row -> stream ->
// position -> page.
#include "attn_dev.h"
#include "paged.h"

namespace xe {
namespace {

constexpr int kT = 256;

struct AppendParams {
  PagedView kv;
  xe_paged_rows r;
  int heads, first;  // heads a row that are written, the first of them (q, then k, then v)
};

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef unsigned u32x2 __attribute__((ext_vector_type(2)));

template <bool VEC>
__device__ __forceinline__ f32x4 load4(const float *p) {
  if constexpr (VEC) return *reinterpret_cast<const f32x4 *>(p);
  else return f32x4{p[0], p[1], p[2], p[3]};
}

__device__ __forceinline__ u32x2 pack_bf16(const f32x4 &x) {
  return u32x2{adev::f32_to_bf16_rne(x[0]) | static_cast<uint32_t>(adev::f32_to_bf16_rne(x[1])) << 16,
               adev::f32_to_bf16_rne(x[2]) | static_cast<uint32_t>(adev::f32_to_bf16_rne(x[3])) << 16};
}

// Stream of row `row`: the last one that starts at or before it, from the
// starts of all streams (empty streams are passed over).  Every thread of the
// block calls it with the same row.
__device__ __forceinline__ int stream_of(const int32_t *start, int batch, int row, int *red) {
  int n = 0;
  for (int j = threadIdx.x; j < batch; j += kT) n += start[j + 1] <= row ? 1 : 0;
#pragma unroll
  for (int off = 32; off >= 1; off >>= 1) n += __shfl_xor(n, off, 64);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = n;
  __syncthreads();
  n = 0;
#pragma unroll
  for (int w = 0; w < kT / 64; w++) n += red[w];
  return n;
}

// hd / 8 lanes take one head of a row: lane l holds dimensions 4 l .. + 3 and
// the four that they are rotated with, hd / 2 further on.
template <int HD, bool VEC>
__global__ __launch_bounds__(kT) void append_kernel(AppendParams p) {
  constexpr int L = HD / 8, HALF = HD / 2, GROUPS = kT / L;
  __shared__ int red[kT / 64];
  const int l = threadIdx.x % L;
  const long long id = static_cast<long long>(blockIdx.x) * GROUPS + threadIdx.x / L;
  const int row0 = static_cast<int>(static_cast<long long>(blockIdx.x) * GROUPS / p.heads);
  const int row = static_cast<int>(id / p.heads), h = p.first + static_cast<int>(id % p.heads);
  int b = row;
  long long pos;
  if (p.r.start) {
    b = stream_of(p.r.start, p.kv.batch, row0, red);
    if (row >= p.r.n_rows) return;
    while (b < p.kv.batch && p.r.start[b + 1] <= row) b++;
    if (b >= p.kv.batch || row < p.r.start[b]) return;  // behind the last stream
    pos = static_cast<long long>(p.r.pos[b]) + (row - p.r.start[b]);
    if (p.r.pos[b] < 0) return;
  } else {
    if (row >= p.r.n_rows) return;
    pos = p.r.pos[b];
  }
  const int page = paged::page_of(p.kv.table + static_cast<size_t>(b) * p.kv.max_pages, p.kv.max_pages, p.kv.n_pages,
                                  p.kv.page_shift, pos);
  if (page < 0 || (p.r.rope_cos && pos >= p.r.rope_len)) return;
  const bool is_q = h < p.r.hq, is_k = !is_q && h < p.r.hq + p.kv.hkv;
  const int kvh = is_k ? h - p.r.hq : h - p.r.hq - p.kv.hkv;
  const float *src = is_q ? p.r.q + static_cast<size_t>(row) * p.r.ldq + h * HD
                          : (is_k ? p.r.k : p.r.v) + static_cast<size_t>(row) * p.r.ldkv + kvh * HD;
  f32x4 x0 = load4<VEC>(src + 4 * l), x1 = load4<VEC>(src + HALF + 4 * l);
  const float *nw = is_q ? p.r.q_norm_w : is_k ? p.r.k_norm_w : nullptr;
  float ss = 0.f;
#pragma unroll
  for (int i = 0; i < 4; i++) ss += x0[i] * x0[i] + x1[i] * x1[i];
  ss = gdev::group_sum(ss, HD == 256 ? 5 : HD == 128 ? 4 : 3);
  if (nw) {
    const float inv = 1.0f / sqrtf(ss / static_cast<float>(HD) + p.r.eps);
#pragma unroll
    for (int i = 0; i < 4; i++) {
      x0[i] = x0[i] * inv * (1.0f + nw[4 * l + i]);
      x1[i] = x1[i] * inv * (1.0f + nw[HALF + 4 * l + i]);
    }
  }
  if (p.r.rope_cos && (is_q || is_k)) {
    const float *cs = p.r.rope_cos + static_cast<size_t>(pos) * HALF + 4 * l;
    const float *sn = p.r.rope_sin + static_cast<size_t>(pos) * HALF + 4 * l;
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const float c = cs[i], s = sn[i], a = x0[i], e = x1[i];
      x0[i] = a * c - e * s;
      x1[i] = e * c + a * s;
    }
  }
  if (is_q) {
    float *dst = p.r.q_out + static_cast<size_t>(row) * p.r.ldqo + h * HD + 4 * l;
    if constexpr (VEC) {
      *reinterpret_cast<f32x4 *>(dst) = x0;
      *reinterpret_cast<f32x4 *>(dst + HALF) = x1;
    } else {
#pragma unroll
      for (int i = 0; i < 4; i++) {
        dst[i] = x0[i];
        dst[HALF + i] = x1[i];
      }
    }
  } else {
    const int slot = static_cast<int>(pos & ((1 << p.kv.page_shift) - 1));
    uint16_t *dst = (is_k ? p.kv.k : p.kv.v) + paged::row_at(p.kv.page_stride, p.kv.page_shift, HD, page, kvh, slot) + 4 * l;
    *reinterpret_cast<u32x2 *>(dst) = pack_bf16(x0);
    *reinterpret_cast<u32x2 *>(dst + HALF) = pack_bf16(x1);
  }
}

template <int HD>
void launch_hd(const AppendParams &p, bool vec, hipStream_t s) {
  constexpr int GROUPS = kT / (HD / 8);
  const long long blocks = (static_cast<long long>(p.r.n_rows) * p.heads + GROUPS - 1) / GROUPS;
  XE_REQUIRE(blocks * kT < (1LL << 32), "paged append: too many rows for one launch");
  hipLaunchKernelGGL((vec ? append_kernel<HD, true> : append_kernel<HD, false>), dim3(static_cast<unsigned>(blocks)),
                     dim3(kT), 0, s, p);
  XE_HIP(hipGetLastError());
}

bool aligned16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

}  // namespace

void launch_paged_append(const PagedView &kv, const xe_paged_rows &r, hipStream_t s) {
  AppendParams p{kv, r, 0, 0};
  p.first = r.q ? 0 : r.hq;
  p.heads = r.hq + 2 * kv.hkv - p.first;
  const bool vec = aligned16(r.k) && aligned16(r.v) && r.ldkv % 4 == 0 &&
                   (!r.q || (aligned16(r.q) && aligned16(r.q_out) && r.ldq % 4 == 0 && r.ldqo % 4 == 0));
  if (kv.hd == 64) launch_hd<64>(p, vec, s);
  else if (kv.hd == 128) launch_hd<128>(p, vec, s);
  else launch_hd<256>(p, vec, s);
}

}  // namespace xe
