// paged_attn.hip -- attention of one new token a stream over the keys and
// values in its pages, split over the streams' lengths and joined.
//
//   out = sum_t softmax(scale q . k_t) v_t over the keys t of the stream
//
// Bound by the bytes of the keys and values: 4 hd a key and kv head against
// 4 hd operations a query head.  What it takes to come near that:
//
// * Shares.  Streams differ in length, so the keys of all units -- (stream,
//   block of up to 16 query heads of a kv head) -- are counted in tiles of 16
//   and shared out equally: few units by whole workgroups, many in one row, from
//   the middle of one unit to the middle of another (below, paged_index.h).  The
//   lengths are on the device, so each workgroup counts them itself.
// * Everything in registers.  A wave takes 16 keys at a time.  Scores come out
//   transposed, S^T = K Q^T (v_mfma_f32_16x16x32_bf16, the keys as A), so a lane
//   holds keys 4 g .. + 3 (g = lane / 16) of query row lane % 16: as they are,
//   the B operand of O^T = V^T P^T (v_mfma_f32_16x16x16_bf16).  For its A operand
//   a lane loads 16 bytes -- 8 dimensions -- of each of these 4 keys, whole rows
//   a load, and turns the block with byte permutes: MFMA e takes dimension 8 n +
//   e as row n.  No LDS for keys and values and no barrier between a unit's
//   first and last key; the next keys load while the values are multiplied, the
//   next values during the next scores, and no load of either hangs on a branch
//   (one that did made every wait one for both: 118 us for 113).
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
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef unsigned u32x2 __attribute__((ext_vector_type(2)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));

constexpr int kTile = 16;    // keys a wave takes at a time, and a granule
constexpr int kRows = 16;    // query heads a unit at most
constexpr int kMaxWg = 512;
constexpr int kGroup = 16;   // partials merged at once
constexpr int kMaxHd = 256;
// Two forms (paged_index.h whole_units): workgroups of eight waves, one a CU,
// whole ones a unit, so that a workgroup has one unit's chain of loads before it;
// else of four waves, two a CU, in equal shares of all keys, with nontemporal loads.
// Those, us plain / nontemporal: 150 mixed streams to 8192 keys (16 / 2 x 128) 113 /
// 103, 48 to 8192 (12 x 64) 159 / 145; 32768 keys of one stream 19.7 / 20.3.
// Equal shares: a unit counts kStart4 tiles on top of its own, about what its
// chain of loads before the first tile and the meeting after the last cost, and
// none is cut within kSlack of its ends.  us without / with: 128 mixed streams
// to 300 keys (12 x 64) 65 / 24, 192 to 5000 (6 / 2 x 64) 51.4 / 46.0; 16 and 16
// take 64 streams to 4096 (4 x 256) from 45.9 to 52.7.
constexpr unsigned kStart4 = 8, kSlack = 8;
static_assert(kSlack >= kStart4, "no share begins among what a unit counts on top");
// Whole workgroups a unit: units of up to kAlone tiles in one workgroup (28
// tiles, 12 units of hd 64: 7.7 us, in two workgroups each 8.9), up to kMore
// tiles a workgroup where a second level of merges is avoided with them (188
// tiles of hd 256: 14.9 us, 15.9 with a tile a workgroup).
constexpr unsigned kAlone = 32, kMore = 24;

__device__ __forceinline__ uint32_t hi16(uint32_t lo, uint32_t hi) { return __builtin_amdgcn_perm(hi, lo, 0x07060302u); }
__device__ __forceinline__ uint32_t lo16(uint32_t lo, uint32_t hi) { return __builtin_amdgcn_perm(hi, lo, 0x05040100u); }
__device__ __forceinline__ float head8(float x) { return __uint_as_float(__float_as_uint(x) & 0xffff0000u); }

// N values as three bf16 parts each, exactly (the upper 8 bits, three times);
// part p of a pair of values in o[p][pair].
template <int N>
__device__ __forceinline__ void parts3(float (&r)[N], uint32_t (&o)[3][N / 2]) {
#pragma unroll
  for (int p = 0; p < 3; p++) {
#pragma unroll
    for (int i = 0; i < N / 2; i++) o[p][i] = hi16(__float_as_uint(r[2 * i]), __float_as_uint(r[2 * i + 1]));
#pragma unroll
    for (int i = 0; i < N; i++) r[i] -= head8(r[i]);
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

// op over the wave, in every lane, and the sum of the lanes up to this one:
// by DPP and lane swaps, without the LDS crossbar.
template <typename Op>
__device__ __forceinline__ unsigned wave_all(unsigned v, Op op) {
  v = op(v, static_cast<unsigned>(gdev::dpp_get_i<gdev::kDppXor1>(static_cast<int>(v))));
  v = op(v, static_cast<unsigned>(gdev::dpp_get_i<gdev::kDppXor2>(static_cast<int>(v))));
  v = op(v, static_cast<unsigned>(gdev::dpp_get_i<gdev::kDppHalfMirror>(static_cast<int>(v))));
  v = op(v, static_cast<unsigned>(gdev::dpp_get_i<gdev::kDppMirror>(static_cast<int>(v))));
  const auto r = __builtin_amdgcn_permlane16_swap(v, v, false, false);
  v = op(r[0], r[1]);
  const auto s = __builtin_amdgcn_permlane32_swap(v, v, false, false);
  return __builtin_amdgcn_readfirstlane(op(s[0], s[1]));
}
template <int CTRL, int ROWS>
__device__ __forceinline__ unsigned add_from(unsigned v) {
  return v + static_cast<unsigned>(__builtin_amdgcn_update_dpp(0, static_cast<int>(v), CTRL, ROWS, 0xF, false));
}
__device__ __forceinline__ unsigned wave_scan(unsigned v) {
  v = add_from<0x111, 0xF>(v);  // row_shr 1, 2, 4, 8: within 16 lanes
  v = add_from<0x112, 0xF>(v);
  v = add_from<0x114, 0xF>(v);
  v = add_from<0x118, 0xF>(v);
  v = add_from<0x142, 0xA>(v);  // lane 15 to the next row
  return add_from<0x143, 0xC>(v);  // lane 31 to the upper half
}

struct Params {
  PagedAttn a;
  float *work;
  unsigned *cnt;
  int group;            // query heads a kv head
  int blocks;           // units of a kv head
  int rows;             // query heads a unit holds room for: min(group, 16)
  unsigned slot_floats; // a partial: O [rows][hd], m [rows], l [rows]
};

constexpr size_t slot_floats_of(int hd, int rows) { return (static_cast<size_t>(rows) * (hd + 2) + 3) & ~size_t(3); }
constexpr int kPad = 4;  // floats between the rows that waves write beside each other
// bytes of the area that holds the queries of a unit, then what its waves found
constexpr size_t area_bytes(int hd, int rows, int kw) {
  const size_t q = static_cast<size_t>(3) * kRows * hd * 2, meet = (static_cast<size_t>(kw) * rows * (hd + kPad) + 2 * kw * kRows) * 4;
  return q > meet ? q : meet;
}

// Partials cross the XCDs' L2s: sc1 stores and loads.
__device__ __forceinline__ void put4(float *base, unsigned idx, const f32x4 &v) {
  __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, v), gdev::coherent_rsrc(base), static_cast<int>(idx * 4), 0,
                                         gdev::kCoherentSc1);
}

template <bool NT, typename P>
__device__ __forceinline__ auto load(P p) {
  if constexpr (NT) return __builtin_nontemporal_load(p);
  else return *p;
}

template <int HD, int KW>
__global__ __launch_bounds__(64 * KW, 2) void paged_attn_kernel(Params p) {
  constexpr int T = 64 * KW;
  constexpr bool kWhole = KW == 8;          // whole workgroups a unit; else equal shares of all keys
  constexpr unsigned kStart = kWhole ? 0 : kStart4;  // granules that a unit counts on top of its own
  constexpr bool kStream = KW == 4;         // keys and values by nontemporal loads
  constexpr int S = HD / 32;                // 32-dimension steps of a score
  constexpr int VB = HD >= 128 ? 8 : 4;     // dimensions of a value a lane loads at once
  constexpr int HV = HD / (16 * VB);        // loads of a value row
  constexpr int NO = HD / 16;               // 16-row blocks of O^T
  typedef unsigned VReg __attribute__((ext_vector_type(VB / 2)));
  extern __shared__ __attribute__((aligned(16))) unsigned char lds[];
  __shared__ unsigned scan[KW + 1];
  __shared__ unsigned found[5];
  unsigned char *const qs = lds;                                              // [3][S][64] x 16 bytes
  float *const meet = reinterpret_cast<float *>(lds);                         // [KW][rows][HD], m and l [KW][kRows]
  int32_t *const lens = reinterpret_cast<int32_t *>(lds + area_bytes(HD, p.rows, KW));  // [batch]
  unsigned *const count = reinterpret_cast<unsigned *>(lens + p.a.kv.batch);            // [batch] granules of a unit

  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const PagedView &kv = p.a.kv;
  const int batch = kv.batch, H = kv.hkv * p.blocks;
  const int cap = kv.max_pages << kv.page_shift;
  const unsigned wg = blockIdx.x, nwg = gridDim.x;

  // Granules of the streams' units: a stream a lane of every wave (kWhole), or
  // some a thread.
  const int each = kWhole ? 1 : (batch + T - 1) / T;
  const int s0 = (kWhole ? lane : tid) * each, s1 = min(s0 + each, batch);  // this thread's streams
  unsigned mine = 0;
  for (int b = s0; b < s1; b++) {
    const int len = p.a.lens[b];
    int lo, hi;
    paged::key_range(len, p.a.window, cap, lo, hi);
    const unsigned n = paged::granules(lo, hi, kTile);
    lens[b] = len;
    count[b] = n;
    mine += n ? n + kStart : 0;
  }
  const unsigned incl = wave_scan(mine * H);
  unsigned before = incl - mine * H, total = __builtin_amdgcn_readlane(incl, 63);
  if constexpr (!kWhole) {
    if (lane == 63) scan[wave] = incl;
    __syncthreads();
    total = 0;
#pragma unroll
    for (int w = 0; w < KW; w++) {
      before += w < wave ? scan[w] : 0u;
      total += scan[w];
    }
    total = __builtin_amdgcn_readfirstlane(total);
  }
  // streams without keys: zeros
  for (int b = wg; b < batch; b += nwg) {
    if (count[b]) continue;
    for (int i = tid; i < p.a.hq * HD; i += T) p.a.out[static_cast<size_t>(b) * p.a.ldo + i] = 0.f;
  }
  if (total == 0) return;

  paged::Div per = paged::div_by(paged::share_of(total, nwg));
  unsigned g0 = wg * per.d;
  unsigned g1 = 0;
  int b = 0;                                   // stream
  unsigned base = 0;                           // its first granule
  unsigned wgs = 0, part = 0, part_unit = 0;   // kWhole: the unit's workgroups, this one among them, the unit
  if constexpr (kWhole) {
    const unsigned units = __popcll(__ballot(mine != 0)) * H;
    const unsigned longest = wave_all(mine, [](unsigned x, unsigned y) { return max(x, y); });
    // the fewest granules a workgroup for which the units' workgroups suffice
    unsigned lo = per.d, hi = nwg > units ? min(longest, paged::share_of(total, nwg - units)) : longest;
    while (lo < hi) {
      const unsigned mid = lo + (hi - lo) / 2;
      if (wave_all(paged::quot_up(mine, paged::div_by(mid)) * H, [](unsigned x, unsigned y) { return x + y; }) <= nwg) hi = mid;
      else lo = mid + 1;
    }
    per = paged::div_by(max(hi, paged::least_share(longest, kGroup, kAlone, kMore)));
    const unsigned own = paged::quot_up(mine, per), upto = wave_scan(own * H);
    const unsigned long long has = __ballot(wg < upto);
    if (!has) return;
    b = __ffsll(has) - 1;
    wgs = __builtin_amdgcn_readlane(own, b);
    const unsigned at = wg - (__builtin_amdgcn_readlane(upto, b) - wgs * H);
    part_unit = at / wgs;
    part = at - part_unit * wgs;
  } else {
    if (g0 >= total) return;
    // where the shares of this workgroup and of the next begin
    if (tid == 0) found[3] = total;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 2; i++) {
      const unsigned g = (wg + i) * per.d;
      if (g < before || g >= before + mine * H) continue;
      unsigned sum = before;
      int s = s0;
      for (;; s++) {
        const unsigned n = count[s] ? (count[s] + kStart) * H : 0;
        if (g < sum + n) break;
        sum += n;
      }
      found[2 + i] = paged::snapped(g, sum, count[s] + kStart, kSlack);
      if (i == 0) {
        found[0] = s;
        found[1] = sum;
      }
    }
    __syncthreads();
    b = __builtin_amdgcn_readfirstlane(found[0]);
    base = __builtin_amdgcn_readfirstlane(found[1]);
    g0 = __builtin_amdgcn_readfirstlane(found[2]);
    g1 = __builtin_amdgcn_readfirstlane(found[3]);
    if (g0 >= g1) return;
  }
  const float sc2 = p.a.scale * adev::kLog2e;
  const size_t head_rows = static_cast<size_t>(1) << kv.page_shift;
  const int slot_mask = (1 << kv.page_shift) - 1;

  for (;;) {
    int own = tid;  // opaque: addresses made from it are not kept over the units
    asm volatile("" : "+v"(own));
    const int ln = own & 15, lg = (own >> 4) & 3;
    int lo, hi;
    paged::key_range(__builtin_amdgcn_readfirstlane(lens[b]), p.a.window, cap, lo, hi);
    const unsigned real = __builtin_amdgcn_readfirstlane(count[b]), n = real ? real + kStart : 0;
    unsigned unit = part_unit, u0 = ~0u, ge = g1;  // partials in slots 2 i + 1
    unsigned w0 = wg - part, nseg = wgs, t0, t1;   // the unit's workgroups, this one's granules of it
    if constexpr (kWhole) {
      paged::part_of(n, wgs, part, t0, t1);
    } else {
      if (g0 >= base + n * H) {
        base += n * H;
        b++;
        continue;
      }
      unit = (g0 - base) / n;
      u0 = base + unit * n;
      ge = min(g1, u0 + n);
      paged::spread(u0, n, per, kSlack, w0, nseg);
      t0 = g0 == u0 ? 0 : g0 - u0 - kStart;
      t1 = ge - u0 - kStart;
    }
    const int kvh = unit / p.blocks, r0 = (unit - kvh * p.blocks) * kRows;
    const int rows = min(p.group - r0, kRows), h0 = kvh * p.group + r0;
    const int first = (lo & ~15) + static_cast<int>(t0) * kTile;
    const int ntile = static_cast<int>(t1 - t0);
    const int32_t *table = kv.table + static_cast<size_t>(b) * kv.max_pages;

    // pages of this wave's next 64 tiles, a tile a lane
    auto pages_from = [&](int i) {
      const int tile = wave + KW * (i + lane);
      return tile < ntile ? paged::page_of(table, kv.max_pages, kv.n_pages, kv.page_shift, first + tile * kTile) : -1;
    };
    int pages = pages_from(0);
    // a lane's part of the queries: row lane % 16 (past the last one: zeros),
    // dimensions 32 s + 8 g .. + 7
    constexpr int SQ = (S + KW - 1) / KW;
    float qx[SQ][8];
    const float *q = p.a.q + static_cast<size_t>(b) * p.a.ldq + static_cast<size_t>(h0 + min(ln, rows - 1)) * HD + 8 * lg;
#pragma unroll
    for (int u = 0; u < SQ; u++)
#pragma unroll
      for (int i = 0; i < 8; i++) qx[u][i] = q[32 * min(wave + KW * u, S - 1) + i];

    u32x4 kr[S];
    VReg vr[4][HV];
    auto row_of = [&](const uint16_t *pool, int i) {  // first key of this wave's tile i
      const int pg = __builtin_amdgcn_readlane(pages, i & 63);
      const int key = first + (wave + KW * i) * kTile;
      return pool + static_cast<size_t>(pg < 0 ? 0 : pg) * kv.page_stride + (kvh * head_rows + (key & slot_mask)) * HD;
    };
    // Past the last tile every lane loads the row's first values again: the
    // number of loads in flight must not depend on a branch, or each wait would
    // be for the keys and the values both.
    const unsigned k_at = (ln * HD + 8 * lg) * 2, v_at = (4 * lg * HD + VB * ln) * 2;  // bytes
    auto load_k = [&](int i, bool more) {
      const char *r = reinterpret_cast<const char *>(row_of(kv.k, i));
      const unsigned at = more ? k_at : 0;
#pragma unroll
      for (int s = 0; s < S; s++) kr[s] = load<kStream>(gptr(reinterpret_cast<const u32x4 *>(r + at + 64 * s)));
    };
    auto load_v = [&](int i, bool more) {
      const char *r = reinterpret_cast<const char *>(row_of(kv.v, i));
      const unsigned at = more ? v_at : 0;
#pragma unroll
      for (int j = 0; j < 4; j++)
#pragma unroll
        for (int c = 0; c < HV; c++) vr[j][c] = load<kStream>(gptr(reinterpret_cast<const VReg *>(r + at + (j * HD + 16 * VB * c) * 2)));
    };

    f32x4 o[NO];
#pragma unroll
    for (int i = 0; i < NO; i++) o[i] = f32x4{0.f, 0.f, 0.f, 0.f};
    float m = -INFINITY, l = 0.f;
    const int tiles = (ntile - wave + KW - 1) / KW;  // this wave's
    load_k(0, tiles > 0);
    load_v(0, tiles > 0);
    // the queries in three parts, operand order, while the first keys load
#pragma unroll
    for (int u = 0; u < SQ; u++) {
      const int s = wave + KW * u;
      uint32_t part[3][4];
#pragma unroll
      for (int i = 0; i < 8; i++) qx[u][i] = ln < rows ? qx[u][i] : 0.f;
      parts3(qx[u], part);
      if (s < S)
#pragma unroll
        for (int i = 0; i < 3; i++)
          *reinterpret_cast<u32x4 *>(qs + ((i * S + s) * 64 + lane) * 16) = u32x4{part[i][0], part[i][1], part[i][2], part[i][3]};
    }
    __syncthreads();
    for (int t = 0; t < tiles; t++) {
      asm volatile("" ::: "memory");  // the queries stay in LDS
      const int key0 = first + (wave + KW * t) * kTile;
      const bool ok = __builtin_amdgcn_readlane(pages, t & 63) >= 0;
      const bool whole = ok && key0 >= lo && key0 + kTile <= hi;
      if ((t & 63) == 63) pages = pages_from(t + 1);
      f32x4 sp[3];  // of each part of the queries: independent chains
#pragma unroll
      for (int i = 0; i < 3; i++) sp[i] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int c = 0; c < S; c++)
#pragma unroll
        for (int i = 0; i < 3; i++)
          sp[i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, kr[c]),
                                                          *reinterpret_cast<const bf16x8 *>(qs + ((i * S + c) * 64 + lane) * 16),
                                                          sp[i], 0, 0, 0);
      const bool more = t + 1 < tiles;
      load_k(more ? t + 1 : t, more);
      float w[4], mb = m;
#pragma unroll
      for (int i = 0; i < 4; i++) {
        w[i] = (sp[0][i] + (sp[1][i] + sp[2][i])) * sc2;
        if (!whole) {
          const int key = key0 + 4 * lg + i;
          w[i] = ok && key >= lo && key < hi ? w[i] : -INFINITY;
        }
        mb = fmaxf(mb, w[i]);
      }
      mb = rows_max(mb);
      const float mu = mb == -INFINITY ? 0.f : mb;  // no key yet: every weight below is exp2(-inf) = 0
      const float corr = __builtin_amdgcn_exp2f(m - mu);
      m = mb;
      l *= corr;
#pragma unroll
      for (int i = 0; i < 4; i++) {
        w[i] = __builtin_amdgcn_exp2f(w[i] - mu);
        l += w[i];
      }
#pragma unroll
      for (int i = 0; i < NO; i++)
#pragma unroll
        for (int j = 0; j < 4; j++) o[i][j] *= corr;
      uint32_t part[3][2];
      parts3(w, part);
      if (!whole) {  // a weight of zero does not silence what is no number
#pragma unroll
        for (int j = 0; j < 4; j++) {
          const int key = key0 + 4 * lg + j;
          const bool on = ok && key >= lo && key < hi;
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
          u32x2 x;
#pragma unroll
          for (int j = 0; j < 2; j++)
            x[j] = (e & 1) ? hi16(vr[2 * j][c][e >> 1], vr[2 * j + 1][c][e >> 1]) : lo16(vr[2 * j][c][e >> 1], vr[2 * j + 1][c][e >> 1]);
#pragma unroll
          for (int i = 0; i < 3; i++)
            o[c * VB + e] = __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(__builtin_bit_cast(s16x4, x),
                                                                      __builtin_bit_cast(s16x4, u32x2{part[i][0], part[i][1]}),
                                                                      o[c * VB + e], 0, 0, 0);
        }
      load_v(more ? t + 1 : t, more);
    }
    l = rows_sum(l);

    // the waves meet
    constexpr int RS = HD + kPad;
    float *const wm = meet + static_cast<size_t>(KW) * p.rows * RS;  // [KW][kRows]
    float *const wl = wm + KW * kRows;
    __syncthreads();  // the queries are done with
    if (lg == 0) {
      wm[wave * kRows + ln] = m;
      wl[wave * kRows + ln] = l;
    }
    if (ln < rows) {
      float *d = meet + (wave * p.rows + ln) * RS + 4 * lg;
#pragma unroll
      for (int i = 0; i < NO; i++) *reinterpret_cast<f32x4 *>(d + 16 * i) = o[i];
    }
    __syncthreads();
    // A head's values lie as the MFMAs left them, here and in partials: value
    // 16 (VB c + e) + k is dimension VB (16 c + k) + e.
    float *const out = p.a.out + static_cast<size_t>(b) * p.a.ldo + static_cast<size_t>(h0) * HD;
    auto finish = [&](int i, f32x4 x, float ls) {
      const int blk = i % HD / 16;
      float *d = out + (i / HD * HD + VB * (16 * (blk / VB) + i % 16) + blk % VB);
      const float inv = ls == 0.f ? 0.f : 1.0f / ls;
#pragma unroll
      for (int z = 0; z < 4; z++) d[VB * z] = ls == 0.f ? 0.f : x[z] * inv;
    };
    const unsigned my_slot = paged::slot_of(u0, per.d, wg) * p.slot_floats;
    for (int i = 4 * own; i < rows * HD; i += 4 * T) {
      const int r = i / HD;
      float mk[KW], mx = -INFINITY, ls = 0.f;
      f32x4 x = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int w = 0; w < KW; w++) mx = fmaxf(mx, mk[w] = wm[w * kRows + r]);
#pragma unroll
      for (int w = 0; w < KW; w++) {
        const float f = mk[w] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(mk[w] - mx);
        const f32x4 v = *reinterpret_cast<const f32x4 *>(meet + ((w * p.rows + r) * RS + i % HD));
        ls += wl[w * kRows + r] * f;
#pragma unroll
        for (int z = 0; z < 4; z++) x[z] += v[z] * f;
      }
      if (nseg == 1) {
        finish(i, x, ls);
      } else {
        put4(p.work, my_slot + i, x);
        if (i % HD == 0) {
          adev::act_st<true>(p.work + my_slot + p.rows * HD + r, mx);
          adev::act_st<true>(p.work + my_slot + p.rows * (HD + 1) + r, ls);
        }
      }
    }
    if (nseg > 1) {
      // Level 0: the partials of this workgroup's group of 16; level 1, and
      // more of them: the groups' first partials, which hold the groups'.
      unsigned seg = wg - w0, left = nseg, step = 1;
      for (;;) {
        const unsigned seg0 = seg / kGroup * kGroup, cnt = min(left - seg0, static_cast<unsigned>(kGroup));
        const bool final = left <= kGroup;
        unsigned *const counter = p.cnt + (step == 1 ? 0 : step == kGroup ? 2 * kMaxWg : 4 * kMaxWg) +
                                  paged::slot_of(u0, per.d, w0 + seg0 * step);
        const bool last = adev::last_to_arrive(counter, static_cast<int>(cnt), reinterpret_cast<int *>(found + 4));
        if (!last) break;
        if (tid == 0) __hip_atomic_store(counter, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        const unsigned dst = paged::slot_of(u0, per.d, w0 + seg0 * step) * p.slot_floats;
        for (int i = 4 * own; i < rows * HD; i += 4 * T) {
          const int r = i / HD;
          float mx = -INFINITY, ls = 0.f;
          f32x4 x = {0.f, 0.f, 0.f, 0.f};
          float mk[kGroup], lk[kGroup];
          f32x4 v[kGroup];
#pragma unroll
          for (int k = 0; k < kGroup; k++) {  // past the last one: that one again, with no weight
            const unsigned sl = paged::slot_of(u0, per.d, w0 + (seg0 + min(static_cast<unsigned>(k), cnt - 1)) * step) * p.slot_floats;
            mk[k] = adev::act_ld<true>(p.work, static_cast<int>(sl + p.rows * HD + r));
            lk[k] = adev::act_ld<true>(p.work, static_cast<int>(sl + p.rows * (HD + 1) + r));
            const float4 t4 = gdev::act_ld4<true>(p.work, static_cast<int>(sl + i));
            v[k] = f32x4{t4.x, t4.y, t4.z, t4.w};
          }
#pragma unroll
          for (int k = 0; k < kGroup; k++) mx = fmaxf(mx, mk[k]);
#pragma unroll
          for (int k = 0; k < kGroup; k++) {
            // A partial without keys holds zeros; one whose scores are all NaN
            // has no maximum either, and its sums have to stay in.
            const float f = mk[k] == -INFINITY || k >= static_cast<int>(cnt) ? 0.f : __builtin_amdgcn_exp2f(mk[k] - mx);
            ls += lk[k] * f;
#pragma unroll
            for (int z = 0; z < 4; z++) x[z] += v[k][z] * f;
          }
          if (final) {
            finish(i, x, ls);
          } else {
            put4(p.work, dst + i, x);
            if (i % HD == 0) {
              adev::act_st<true>(p.work + dst + p.rows * HD + r, mx);
              adev::act_st<true>(p.work + dst + p.rows * (HD + 1) + r, ls);
            }
          }
        }
        if (final) break;
        seg /= kGroup;
        left = (left + kGroup - 1) / kGroup;
        step *= kGroup;
      }
    }
    g0 = ge;
    if (kWhole || g0 >= g1) break;
    __syncthreads();  // the area is free again
  }
}

using PagedFn = void (*)(Params);
template <int KW>
PagedFn pick(int hd) {
  return hd == 64 ? paged_attn_kernel<64, KW> : hd == 128 ? paged_attn_kernel<128, KW> : paged_attn_kernel<256, KW>;
}

}  // namespace

size_t paged_work_floats() { return static_cast<size_t>(2) * kMaxWg * slot_floats_of(kMaxHd, kRows); }
size_t paged_cnt_words() { return static_cast<size_t>(6) * kMaxWg; }

void launch_paged_attn(const PagedAttn &a, float *work, unsigned *cnt, hipStream_t s) {
  Params p{a, work, cnt, a.hq / a.kv.hkv, 0, 0, 0};
  p.blocks = (p.group + kRows - 1) / kRows;
  p.rows = std::min(p.group, kRows);
  p.slot_floats = static_cast<unsigned>(slot_floats_of(a.kv.hd, p.rows));
  const int64_t cap = static_cast<int64_t>(a.kv.max_pages) << a.kv.page_shift;
  const int64_t units = static_cast<int64_t>(a.kv.batch) * a.kv.hkv * p.blocks;
  XE_REQUIRE(cap / kTile * units < (int64_t(1) << 31), "paged attention: more than 2^31 blocks of 16 keys in the table");
  const int64_t span = a.window ? std::min<int64_t>(cap, static_cast<int64_t>(a.window) + kTile) : cap;
  const bool wide = paged::whole_units(a.kv.batch, units, span, a.kv.hd, gdev::cu_count());
  const int kw = wide ? 8 : 4;
  const int64_t wgs = std::max<int64_t>(1, std::min<int64_t>(std::min(kMaxWg, (wide ? 1 : 2) * gdev::cu_count()), cap / kTile * units));
  const size_t lds = area_bytes(a.kv.hd, p.rows, kw) + 8 * static_cast<size_t>(a.kv.batch);
  const PagedFn fn = wide ? pick<8>(a.kv.hd) : pick<4>(a.kv.hd);
  if (lds > 64 * 1024)
    XE_HIP(hipFuncSetAttribute(reinterpret_cast<const void *>(fn), hipFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(lds)));
  hipLaunchKernelGGL(fn, dim3(static_cast<unsigned>(wgs)), dim3(64 * kw), lds, s, p);
  XE_HIP(hipGetLastError());
}

}  // namespace xe
