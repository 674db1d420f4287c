// paged_attn.hip -- attention of one new token a stream over the keys and
// values in its pages, split over the streams' lengths and joined.
//
//   out = sum_t softmax(scale q . k_t) v_t over the keys t of the stream
//
// Bound by the bytes of the keys and values: 4 hd a key and kv head against
// 4 hd operations a query head.  What it takes to come near that:
//
// * Equal shares.  Streams differ in length, so the keys of all (stream,
//   block of up to 16 query heads of a kv head) units are cut into granules of
//   256 keys, and every workgroup takes the same number of granules in a row,
//   from the middle of one unit to the middle of another (paged_index.h).  The
//   lengths are on the device, so each workgroup sums them up itself.
// * Everything in registers.  A wave takes 32 keys at a time.  Scores come out
//   transposed, S^T = K Q^T (v_mfma_f32_16x16x32_bf16, 16 keys as A), so a lane
//   holds keys 4 g .. + 3 (g = lane / 16) of query row lane % 16: as they are,
//   the B operand of O^T = V^T P^T with k slot 8 g + j read as key 4 g + j of
//   the first 16 keys (j < 4) or of the second.  For its A operand a lane loads
//   16 bytes -- 8 dimensions -- of each of its 8 keys, whole rows a load, and
//   turns the 8 x 8 block with byte permutes: MFMA e takes dimension 8 n + e as
//   row n.  No LDS and no barrier between a unit's first and last key; the next
//   keys load while the values are multiplied, the next values during the next
//   scores.
// * fp32 results.  Queries and probabilities are three bf16 parts each, exact
//   (8 bits a part); keys and values are bf16 as stored; scores, softmax
//   statistics and sums are fp32, the softmax with a running maximum, base 2.
// * One launch.  A unit that one workgroup holds whole is written out; the
//   others leave partials (m, l, O), and the last workgroup of 16 to arrive
//   merges theirs, the last of these groups the groups'.  The order of every
//   sum is that of the keys, whoever arrives last.
#include <algorithm>

#include "attn_dev.h"
#include "paged.h"

namespace xe {
namespace {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef unsigned u32x2 __attribute__((ext_vector_type(2)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));

constexpr int kW = 8;                // waves a workgroup
constexpr int kT = 64 * kW;
constexpr int kTile = 32;            // keys a wave takes at a time
constexpr int kGranule = kTile * kW; // keys a workgroup takes at a time
constexpr int kRows = 16;            // query heads a unit at most
constexpr int kMaxWg = 512;
constexpr int kGroup = 16;           // partials merged at once
constexpr int kMaxMerge = kMaxWg / kGroup + 1;

__device__ __forceinline__ uint32_t hi16(uint32_t lo, uint32_t hi) { return __builtin_amdgcn_perm(hi, lo, 0x07060302u); }
__device__ __forceinline__ uint32_t lo16(uint32_t lo, uint32_t hi) { return __builtin_amdgcn_perm(hi, lo, 0x05040100u); }
__device__ __forceinline__ float head8(float x) { return __uint_as_float(__float_as_uint(x) & 0xffff0000u); }

// v = sum of three bf16 parts, exactly (the upper 8 bits, three times).
__device__ __forceinline__ void parts3(const float (&v)[8], bf16x8 (&o)[3]) {
  float r[8];
#pragma unroll
  for (int i = 0; i < 8; i++) r[i] = v[i];
#pragma unroll
  for (int p = 0; p < 3; p++) {
    u32x4 w;
#pragma unroll
    for (int i = 0; i < 4; i++) w[i] = hi16(__float_as_uint(r[2 * i]), __float_as_uint(r[2 * i + 1]));
    o[p] = __builtin_bit_cast(bf16x8, w);
#pragma unroll
    for (int i = 0; i < 8; i++) r[i] -= head8(r[i]);
  }
}

// The largest / the sum over the four lanes of a query row (lane % 16).
__device__ __forceinline__ float rows_max(float v) {
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
  const auto s = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(s[0]), __uint_as_float(s[1]));
}
__device__ __forceinline__ float rows_sum(float v) {
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = __uint_as_float(r[0]) + __uint_as_float(r[1]);
  const auto s = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(s[0]) + __uint_as_float(s[1]);
}

struct Params {
  PagedAttn a;
  float *work;
  unsigned *cnt;
  int group;       // query heads a kv head
  int blocks;      // units of a kv head
  int rows;        // query heads a unit holds room for: min(group, 16)
  unsigned least;  // granules a workgroup takes at least
};

template <int HD>
constexpr size_t q_bytes() {
  return static_cast<size_t>(3) * kRows * HD * 2;
}
// floats of the area where a workgroup's waves, or partials, meet
constexpr size_t meet_floats(int hd, int rows) {
  return static_cast<size_t>(kW) * rows * hd + 2 * kW * kRows + kRows * kMaxMerge + 2 * kRows;
}

template <int HD>
__global__ __launch_bounds__(kT) void paged_attn_kernel(Params p) {
  constexpr int S = HD / 32;                // 32-dimension steps of a score
  constexpr int VB = HD >= 128 ? 8 : 4;     // dimensions of a value a lane loads at once
  constexpr int HV = HD / (16 * VB);        // loads of a value row
  constexpr int NO = HD / 16;               // 16-row blocks of O^T
  typedef unsigned VReg __attribute__((ext_vector_type(VB / 2)));
  extern __shared__ __attribute__((aligned(16))) unsigned char lds[];
  int32_t *const lens = reinterpret_cast<int32_t *>(lds);                        // [batch]
  unsigned char *const area = lds + ((4 * p.a.kv.batch + 15) & ~15);
  unsigned char *const qs = area;                                                // [3][S][64] x 16 bytes
  float *const meet = reinterpret_cast<float *>(area);                           // after a unit's last key
  __shared__ unsigned scan[kW + 1];
  __shared__ unsigned found[4];

  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int ln = lane & 15, lg = lane >> 4;
  const PagedView &kv = p.a.kv;
  const int batch = kv.batch, H = kv.hkv * p.blocks;
  const int cap = kv.max_pages << kv.page_shift;
  const unsigned wg = blockIdx.x, nwg = gridDim.x;

  // granules of the streams: this thread's, the sum before them, all of them
  const int per_thread = (batch + kT - 1) / kT;
  unsigned mine = 0;
  for (int i = 0; i < per_thread; i++) {
    const int b = tid * per_thread + i;
    if (b >= batch) break;
    const int len = p.a.lens[b];
    lens[b] = len;
    int lo, hi;
    paged::key_range(len, p.a.window, cap, lo, hi);
    mine += paged::granules(lo, hi, kGranule) * H;
  }
  unsigned incl = mine;
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) {
    const unsigned o = __shfl_up(incl, off, 64);
    if (lane >= off) incl += o;
  }
  if (lane == 63) scan[wave] = incl;
  if (tid == 0) found[0] = batch;
  __syncthreads();
  unsigned before = incl - mine, total = 0;
#pragma unroll
  for (int w = 0; w < kW; w++) {
    before += w < wave ? scan[w] : 0u;
    total += scan[w];
  }
  // streams without keys: zeros
  for (int b = wg; b < batch; b += nwg) {
    int lo, hi;
    paged::key_range(lens[b], p.a.window, cap, lo, hi);
    if (hi > lo) continue;
    for (int i = tid; i < p.a.hq * HD; i += kT) p.a.out[static_cast<size_t>(b) * p.a.ldo + i] = 0.f;
  }
  if (total == 0) return;
  const unsigned per = paged::share_of(total, nwg, p.least);
  unsigned g0 = wg * per;
  const unsigned g1 = min(g0 + per, total);
  if (g0 >= total) return;
  if (g0 >= before && g0 < before + mine) {  // the stream of the first granule
    unsigned at = before;
    int b = tid * per_thread;
    for (;; b++) {
      int lo, hi;
      paged::key_range(lens[b], p.a.window, cap, lo, hi);
      const unsigned n = paged::granules(lo, hi, kGranule) * H;
      if (g0 < at + n) break;
      at += n;
    }
    found[0] = b;
    found[1] = at;
  }
  __syncthreads();
  int b = found[0];
  unsigned base = found[1];  // first granule of stream b
  const float sc2 = p.a.scale * adev::kLog2e;

  while (g0 < g1) {
    int lo, hi;
    paged::key_range(lens[b], p.a.window, cap, lo, hi);
    const unsigned n = paged::granules(lo, hi, kGranule);
    if (g0 >= base + n * H) {
      base += n * H;
      b++;
      continue;
    }
    const unsigned unit = (g0 - base) / n, u0 = base + unit * n, u1 = u0 + n;
    const unsigned ge = min(g1, u1);  // this workgroup's granules of the unit: [g0, ge)
    const int kvh = unit / p.blocks, r0 = (unit % p.blocks) * kRows;
    const int rows = min(p.group - r0, kRows), h0 = kvh * p.group + r0;
    const int first = (lo & ~15) + static_cast<int>(g0 - u0) * kGranule;
    const int end = min(hi, first + static_cast<int>(ge - g0) * kGranule);
    const int32_t *table = kv.table + static_cast<size_t>(b) * kv.max_pages;

    // pages of this wave's next 32 tiles, one 16-key block a lane
    auto pages_from = [&](int tile) {
      const int key = first + (wave + kW * (tile + (lane >> 1))) * kTile + 16 * (lane & 1);
      return key < end ? paged::page_of(table, kv.max_pages, kv.n_pages, kv.page_shift, key) : -1;
    };
    int pages = pages_from(0);

    // queries in three parts, operand order
    for (int s = wave; s < S; s += kW) {
      float x[8];
      const float *q = p.a.q + static_cast<size_t>(b) * p.a.ldq + static_cast<size_t>(h0 + ln) * HD + 32 * s + 8 * lg;
#pragma unroll
      for (int i = 0; i < 8; i++) x[i] = ln < rows ? q[i] : 0.f;
      bf16x8 o[3];
      parts3(x, o);
#pragma unroll
      for (int i = 0; i < 3; i++) *reinterpret_cast<bf16x8 *>(qs + ((i * S + s) * 64 + lane) * 16) = o[i];
    }
    __syncthreads();

    u32x4 kr[2][S];
    VReg vr[8][HV];
    const size_t head = static_cast<size_t>(kvh) << kv.page_shift;
    const int slot_mask = (1 << kv.page_shift) - 1;
    auto at_block = [&](const uint16_t *pool, int tile, int blk) {  // row of the block's first key
      const int pg = __builtin_amdgcn_readlane(pages, 2 * (tile & 31) + blk);
      const int key = first + (wave + kW * tile) * kTile + 16 * blk;
      return pool + static_cast<size_t>(pg < 0 ? 0 : pg) * kv.page_stride + (head + (key & slot_mask)) * HD;
    };
    auto load_k = [&](int tile) {
#pragma unroll
      for (int q = 0; q < 2; q++) {
        const uint16_t *r = at_block(kv.k, tile, q) + ln * HD + 8 * lg;
#pragma unroll
        for (int s = 0; s < S; s++) kr[q][s] = *gptr(reinterpret_cast<const u32x4 *>(r + 32 * s));
      }
    };
    auto load_v = [&](int tile) {
#pragma unroll
      for (int q = 0; q < 2; q++) {
        const uint16_t *r = at_block(kv.v, tile, q) + 4 * lg * HD + VB * ln;
#pragma unroll
        for (int j = 0; j < 4; j++)
#pragma unroll
          for (int c = 0; c < HV; c++) vr[4 * q + j][c] = *gptr(reinterpret_cast<const VReg *>(r + j * HD + 16 * VB * c));
      }
    };

    f32x4 o[NO];
#pragma unroll
    for (int i = 0; i < NO; i++) o[i] = f32x4{0.f, 0.f, 0.f, 0.f};
    float m = -INFINITY, l = 0.f;
    const int tiles = (end - first + kTile * kW - 1 - wave * kTile) / (kTile * kW);  // this wave's
    if (tiles > 0) {
      load_k(0);
      load_v(0);
    }
    for (int t = 0; t < tiles; t++) {
      const int key0 = first + (wave + kW * t) * kTile;
      const bool ok0 = __builtin_amdgcn_readlane(pages, 2 * (t & 31)) >= 0;
      const bool ok1 = __builtin_amdgcn_readlane(pages, 2 * (t & 31) + 1) >= 0;
      const bool whole = ok0 && ok1 && key0 >= lo && key0 + kTile <= end;
      if ((t & 31) == 31 && t + 1 < tiles) pages = pages_from(t + 1);
      if constexpr (HD == 256) asm volatile("" ::: "memory");  // the queries stay in LDS: 96 registers
      f32x4 s[2] = {f32x4{0.f, 0.f, 0.f, 0.f}, f32x4{0.f, 0.f, 0.f, 0.f}};
#pragma unroll
      for (int c = 0; c < S; c++)
#pragma unroll
        for (int i = 0; i < 3; i++) {
          const bf16x8 q = *reinterpret_cast<const bf16x8 *>(qs + ((i * S + c) * 64 + lane) * 16);
#pragma unroll
          for (int k = 0; k < 2; k++)
            s[k] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, kr[k][c]), q, s[k], 0, 0, 0);
        }
      if (t + 1 < tiles) load_k(t + 1);
      float mb = m;
#pragma unroll
      for (int k = 0; k < 2; k++)
#pragma unroll
        for (int i = 0; i < 4; i++) {
          s[k][i] *= sc2;
          if (!whole) {
            const int key = key0 + 16 * k + 4 * lg + i;
            s[k][i] = (k ? ok1 : ok0) && key >= lo && key < end ? s[k][i] : -INFINITY;
          }
          mb = fmaxf(mb, s[k][i]);
        }
      mb = rows_max(mb);
      const float mu = mb == -INFINITY ? 0.f : mb;  // no key yet: every weight below is exp2(-inf) = 0
      const float corr = __builtin_amdgcn_exp2f(m - mu);
      m = mb;
      float w[8];
      l *= corr;
#pragma unroll
      for (int i = 0; i < 8; i++) {
        w[i] = __builtin_amdgcn_exp2f(s[i >> 2][i & 3] - mu);
        l += w[i];
      }
#pragma unroll
      for (int i = 0; i < NO; i++)
#pragma unroll
        for (int j = 0; j < 4; j++) o[i][j] *= corr;
      bf16x8 pf[3];
      parts3(w, pf);
      if (!whole) {  // a weight of zero does not silence what is no number
#pragma unroll
        for (int j = 0; j < 8; j++) {
          const int key = key0 + 16 * (j >> 2) + 4 * lg + (j & 3);
          const bool on = ((j >> 2) ? ok1 : ok0) && key >= lo && key < end;
#pragma unroll
          for (int c = 0; c < HV; c++)
#pragma unroll
            for (int e = 0; e < VB / 2; e++) vr[j][c][e] = on ? vr[j][c][e] : 0u;
        }
      }
#pragma unroll
      for (int c = 0; c < HV; c++)
#pragma unroll
        for (int e = 0; e < VB; e++) {
          u32x4 x;
#pragma unroll
          for (int j = 0; j < 4; j++)
            x[j] = (e & 1) ? hi16(vr[2 * j][c][e >> 1], vr[2 * j + 1][c][e >> 1]) : lo16(vr[2 * j][c][e >> 1], vr[2 * j + 1][c][e >> 1]);
          const bf16x8 vf = __builtin_bit_cast(bf16x8, x);
#pragma unroll
          for (int i = 0; i < 3; i++)
            o[c * VB + e] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vf, pf[i], o[c * VB + e], 0, 0, 0);
        }
      if (t + 1 < tiles) load_v(t + 1);
    }
    l = rows_sum(l);

    // the waves meet: (m, l) and O of each
    float *const wm = meet + static_cast<size_t>(kW) * p.rows * HD;  // [kW][kRows]
    float *const wl = wm + kW * kRows;
    float *const fac = wl + kW * kRows;  // [kRows][kMaxMerge] weights of what is merged
    float *const ml = fac + kRows * kMaxMerge;
    __syncthreads();  // the queries are done with
    if (lg == 0) {
      wm[wave * kRows + ln] = m;
      wl[wave * kRows + ln] = l;
    }
    if (ln < rows) {
      float *d = meet + (static_cast<size_t>(wave) * p.rows + ln) * HD;
#pragma unroll
      for (int c = 0; c < HV; c++)
#pragma unroll
        for (int i = 0; i < 4; i++)
#pragma unroll
          for (int e = 0; e < VB; e += 4) {  // lane (4 g + i) of block e holds dimension VB (4 g + i) + e
            f32x4 x;
#pragma unroll
            for (int z = 0; z < 4; z++) x[z] = o[c * VB + e + z][i];
            *reinterpret_cast<f32x4 *>(d + c * 16 * VB + VB * (4 * lg + i) + e) = x;
          }
    }
    __syncthreads();
    if (tid < kRows) {
      float mx = -INFINITY, ls = 0.f;
#pragma unroll
      for (int w = 0; w < kW; w++) mx = fmaxf(mx, wm[w * kRows + tid]);
#pragma unroll
      for (int w = 0; w < kW; w++) {
        const float f = wm[w * kRows + tid] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(wm[w * kRows + tid] - mx);
        fac[tid * kMaxMerge + w] = f;
        ls += wl[w * kRows + tid] * f;
      }
      ml[2 * tid] = mx;
      ml[2 * tid + 1] = ls;
    }
    __syncthreads();
    const unsigned w0 = paged::first_wg(u0, per), nseg = paged::wg_count(u0, u1, per);
    const size_t slot_floats = static_cast<size_t>(p.rows) * (HD + 2);
    float *const out = p.a.out + static_cast<size_t>(b) * p.a.ldo + static_cast<size_t>(h0) * HD;
    float *const part = p.work + paged::slot_of(u0, per, wg) * slot_floats;
    for (int i = tid; i < rows * HD; i += kT) {
      const int r = i / HD;
      float x = 0.f;
#pragma unroll
      for (int w = 0; w < kW; w++) x += meet[static_cast<size_t>(w) * p.rows * HD + i] * fac[r * kMaxMerge + w];
      if (nseg == 1) {
        const float ls = ml[2 * r + 1];
        out[i] = ls == 0.f ? 0.f : x / ls;
      } else {
        adev::act_st<true>(part + 2 * p.rows + i, x);
      }
    }
    if (nseg > 1) {
      if (tid < 2 * rows) adev::act_st<true>(part + tid, ml[tid]);
      // merges n partials, the one after i in slot(i), over part 0 or to out
      auto merge = [&](unsigned cnt, auto slot, bool final) {
        const float *const w = p.work;
        for (int i = tid; i < rows * kMaxMerge; i += kT) {
          const int r = i / kMaxMerge;
          const unsigned k = i % kMaxMerge;
          if (k < cnt) {
            const int at = static_cast<int>(slot(k) * slot_floats) + 2 * r;
            meet[i] = adev::act_ld<true>(w, at);
            fac[i] = adev::act_ld<true>(w, at + 1);
          }
        }
        __syncthreads();
        if (tid < rows) {
          float mx = -INFINITY, ls = 0.f;
          for (unsigned k = 0; k < cnt; k++) mx = fmaxf(mx, meet[tid * kMaxMerge + k]);
          for (unsigned k = 0; k < cnt; k++) {
            const float mk = meet[tid * kMaxMerge + k];
            const float f = mk == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(mk - mx);
            ls += fac[tid * kMaxMerge + k] * f;
            fac[tid * kMaxMerge + k] = f;
          }
          ml[2 * tid] = mx;
          ml[2 * tid + 1] = ls;
        }
        __syncthreads();
        for (int i = tid; i < rows * HD; i += kT) {
          const int r = i / HD;
          float x = 0.f;
          for (unsigned k0 = 0; k0 < cnt; k0 += kGroup) {
            float v[kGroup];
#pragma unroll
            for (int k = 0; k < kGroup; k++)
              v[k] = k0 + k < cnt ? adev::act_ld<true>(w, static_cast<int>(slot(k0 + k) * slot_floats) + 2 * p.rows + i) : 0.f;
#pragma unroll
            for (int k = 0; k < kGroup; k++)
              if (k0 + k < cnt) x += v[k] * fac[r * kMaxMerge + k0 + k];
          }
          if (final) {
            const float ls = ml[2 * r + 1];
            out[i] = ls == 0.f ? 0.f : x / ls;
          } else {
            adev::act_st<true>(p.work + slot(0) * slot_floats + 2 * p.rows + i, x);
          }
        }
        if (!final && tid < 2 * rows) adev::act_st<true>(p.work + slot(0) * slot_floats + tid, ml[tid]);
      };
      auto arrive = [&](unsigned *cnt, unsigned n) {  // whether this workgroup is the last of n
        const bool last = adev::last_to_arrive(cnt, static_cast<int>(n), reinterpret_cast<int *>(found + 2));
        if (last && tid == 0) __hip_atomic_store(cnt, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        return last;
      };
      const unsigned grp = (wg - w0) / kGroup, groups = (nseg + kGroup - 1) / kGroup;
      const unsigned in_grp = min(nseg - grp * kGroup, static_cast<unsigned>(kGroup));
      auto seg_slot = [&](unsigned seg) { return paged::slot_of(u0, per, w0 + seg); };
      if (arrive(p.cnt + seg_slot(grp * kGroup), in_grp)) {
        merge(in_grp, [&](unsigned k) { return seg_slot(grp * kGroup + k); }, groups == 1);
        if (groups > 1 && arrive(p.cnt + 2 * kMaxWg + seg_slot(0), groups))
          merge(groups, [&](unsigned k) { return seg_slot(k * kGroup); }, true);
      }
    }
    __syncthreads();  // the area is free again
    g0 = ge;
  }
}

}  // namespace

size_t paged_work_floats() { return static_cast<size_t>(2) * kMaxWg * kRows * (256 + 2); }
size_t paged_cnt_words() { return static_cast<size_t>(4) * kMaxWg; }

void launch_paged_attn(const PagedAttn &a, float *work, unsigned *cnt, hipStream_t s) {
  Params p{a, work, cnt, a.hq / a.kv.hkv, 0, 0, 1};
  p.blocks = (p.group + kRows - 1) / kRows;
  p.rows = std::min(p.group, kRows);
  const int64_t cap = static_cast<int64_t>(a.kv.max_pages) << a.kv.page_shift;
  const int64_t most = (cap + kGranule - 1) / kGranule * a.kv.batch * a.kv.hkv * p.blocks;
  XE_REQUIRE(most < (int64_t(1) << 31), "paged attention: more than 2^31 blocks of keys in the table");
  const int64_t all = std::max<int64_t>(1, std::min<int64_t>(kMaxWg, most));
  const size_t area = std::max(static_cast<size_t>(3) * kRows * a.kv.hd * 2, meet_floats(a.kv.hd, p.rows) * sizeof(float));
  const size_t lds = ((4 * static_cast<size_t>(a.kv.batch) + 15) & ~size_t(15)) + area;
  auto fn = a.kv.hd == 64 ? paged_attn_kernel<64> : a.kv.hd == 128 ? paged_attn_kernel<128> : paged_attn_kernel<256>;
  if (lds > 64 * 1024)
    XE_HIP(hipFuncSetAttribute(reinterpret_cast<const void *>(fn), hipFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(lds)));
  hipLaunchKernelGGL(fn, dim3(static_cast<unsigned>(all)), dim3(kT), lds, s, p);
  XE_HIP(hipGetLastError());
}

}  // namespace xe
