"""Paged cache, host side (CPU): the arithmetic that finds a key's page, over
bad tables and positions, and what the entry points refuse."""
import ctypes as C
import os
import shutil
import subprocess

import pytest

from conftest import ROOT, load_xe

CSRC = os.path.join(ROOT, "xdna-engine_amd", "csrc")


class At:
    def __init__(self, ptr):
        self.ptr = ptr


@pytest.fixture(scope="module")
def xe():
    return load_xe()


@pytest.fixture
def kv(xe):
    return xe.PagedKV(At(0x1000), At(0x2000), At(0x3000), 8, 2, 16, 64, 3, 4)


@pytest.fixture
def rows(xe):
    return xe.PagedRows(3, 4, q=0x4000, k=0x5000, v=0x6000, ldq=256, ldkv=128, q_out=0x7000, ldqo=256, pos=0x8000)


def test_page_arithmetic(tmp_path):
    """Every page that page_of gives is in the pool, every offset of row_at in
    its page, also beyond 2^32 elements; key ranges are ordered and in the table."""
    if shutil.which("g++") is None:
        pytest.skip("no g++")
    src = tmp_path / "t.cpp"
    src.write_text(r'''
#include "paged_index.h"
#include <cassert>
#include <climits>
#include <vector>
using namespace xe::paged;
int main() {
  const int32_t row[4] = {5, -1, 8, INT_MAX};
  assert(page_of(row, 4, 8, 4, 0) == 5 && page_of(row, 4, 8, 4, 15) == 5);
  for (long long p = 16; p < 80; p++) assert(page_of(row, 4, 8, 4, p) == -1);
  assert(page_of(row, 4, 9, 4, 32) == 8);
  assert(page_of(row, 4, 8, 4, -1) == -1 && page_of(row, 4, 8, 4, LLONG_MAX) == -1 && page_of(row, 4, 8, 4, 1LL << 32) == -1);
  const size_t stride = (size_t)12 * 1024 * 256;
  assert(row_at(stride, 10, 256, 100000, 11, 1023) == (size_t)100000 * stride + (size_t)(11 * 1024 + 1023) * 256);
  assert(row_at(stride, 10, 256, 0, 11, 1023) + 256 == stride);
  for (int len : {INT_MIN, -1, 0, 1, 15, 16, 17, 63, 64, 65, 1000, INT_MAX})
    for (int window : {0, 1, 16, 64, 65, INT_MAX})
      for (int cap : {16, 64, 1 << 30}) {
        int lo, hi;
        key_range(len, window, cap, lo, hi);
        assert(0 <= lo && lo <= hi);
        assert(hi == lo || hi <= cap);
        const long long n = len < 0 ? 0 : len;
        const long long first = window && n > window ? n - window : 0, last = n < cap ? n : cap;
        assert((long long)hi - lo == (last > first ? last - first : 0));
        assert(hi == lo || lo == first);
      }
}
''')
    exe = str(tmp_path / "t")
    subprocess.check_call(["g++", "-std=c++17", "-fsanitize=undefined,address", "-I" + CSRC, str(src), "-o", exe])
    subprocess.check_call([exe], timeout=60)


def test_shares(tmp_path):
    """Every granule belongs to exactly one workgroup, each workgroup's partials
    to places of their own, and a unit's partials are found where they lie."""
    if shutil.which("g++") is None:
        pytest.skip("no g++")
    src = tmp_path / "s.cpp"
    src.write_text(r'''
#include "paged_index.h"
#include <cassert>
#include <random>
#include <set>
#include <vector>
using namespace xe::paged;
int main() {
  std::mt19937 rng(3);
  auto pick = [&](int n) { return (int)(rng() % n); };
  assert(granules(0, 0, 256) == 0 && granules(5, 6, 256) == 1 && granules(0, 256, 256) == 1 && granules(0, 257, 256) == 2);
  assert(granules(15, 256, 256) == 1 && granules(17, 272, 256) == 1 && granules(17, 273, 256) == 2);
  for (int round = 0; round < 3000; round++) {
    const int units = 1 + pick(40), most = 1 << pick(10);
    std::vector<unsigned> n(units);
    unsigned total = 0;
    for (auto &x : n) total += x = pick(3) ? 1 + pick(most) : 1;
    const unsigned nwg = pick(2) ? 256 : 1 + pick(512), per = share_of(total, nwg);
    const Div by = div_by(per);
    assert(per >= 1 && (unsigned long long)per * nwg >= total);
    const unsigned slack = pick(3) ? pick(20) : pick(200);
    std::vector<unsigned> begin(nwg + 1, total);  // of each share
    {
      unsigned u0 = 0, i = 0;
      for (int u = 0; u < units; u0 += n[u++])
        for (; i <= nwg && i * per < u0 + n[u]; i++) begin[i] = snapped(i * per, u0, n[u], slack);
      for (unsigned k = 0; k < nwg; k++) assert(begin[k] <= begin[k + 1]);
      assert(begin[0] == 0 && begin[nwg] == total);
    }
    std::set<unsigned> places;
    unsigned u0 = 0, covered = 0;
    for (int u = 0; u < units; u++) {
      const unsigned u1 = u0 + n[u];
      unsigned w0 = ~0u, cnt = 0, has = 0, first = 0;
      for (unsigned wg = 0; wg < nwg; wg++) {
        const unsigned a = begin[wg] > u0 ? begin[wg] : u0, z = begin[wg + 1] < u1 ? begin[wg + 1] : u1;
        if (a >= z) continue;
        if (!has++) first = wg;
        assert(wg == first + has - 1);
        covered += z - a;
      }
      spread(u0, n[u], by, slack, w0, cnt);
      assert(cnt == has);
      if (cnt > 1) {
        assert(w0 == first && w0 + cnt <= nwg);
        for (unsigned wg = w0; wg < w0 + cnt; wg++) {
          const unsigned slot = slot_of(u0, per, wg);
          assert(slot < 2 * nwg && places.insert(slot).second);
        }
      }
      u0 = u1;
    }
    assert(covered == total);
    for (int u = 0; u < units; u++) {  // whole workgroups
      const unsigned wgs = quot_up(n[u], by);
      unsigned upto = 0, most = 0, least = ~0u;
      for (unsigned i = 0; i < wgs; i++) {
        unsigned t0, t1;
        part_of(n[u], wgs, i, t0, t1);
        assert(t0 == upto && t1 > t0 && t1 - t0 <= per);
        upto = t1;
        most = t1 - t0 > most ? t1 - t0 : most;
        least = t1 - t0 < least ? t1 - t0 : least;
      }
      assert(upto == n[u] && most - least <= 1);
    }
  }
  for (int round = 0; round < 300000; round++) {
    unsigned a = rng(), d = rng() >> (rng() % 32);
    if (round % 7 == 0) a = ~0u - pick(3);
    if (round % 5 == 0) a = (a / (d ? d : 1)) * (d ? d : 1) - pick(2);
    if (d == 0) d = 1;
    assert(quot(a, div_by(d)) == a / d && quot_up(a, div_by(d)) == a / d + (a % d != 0));
  }
}
''')
    exe = str(tmp_path / "s")
    subprocess.check_call(["g++", "-O1", "-std=c++17", "-fsanitize=undefined,address", "-I" + CSRC, str(src), "-o", exe])
    subprocess.check_call([exe], timeout=60)


def test_forms_of_the_rows_product(tmp_path):
    """Every form is taken by some shape, by one of those that the GPU tests run
    among them, and none whose partial tiles do not fit the workspace."""
    if shutil.which("g++") is None:
        pytest.skip("no g++")
    src = tmp_path / "f.cpp"
    src.write_text(r'''
#include "rows_form.h"
#include <cassert>
#include <initializer_list>
using namespace xe::rowsform;
int main() {
  int seen[kForms] = {};
  for (int m : {1, 15, 16, 100, 1000, 4096, 14336, 65536, 1000000, 134217727})
    for (int k : {16, 64, 1152, 4096, 16384, 32768})
      for (int batch : {1, 2, 3, 16, 33, 64, 65, 200, 511, 512})
        for (int cus : {1, 64, 256, 304}) {
          const int i = pick(m, k, batch, cus);
          assert(i >= 0 && i < kForms && fits(i, m, batch));
        }
  for (int i = 0; i < kForms; i++)
    if (kForm[i].ksplit > 1) {
      assert(fits(i, kForm[i].bm, kForm[i].bn) && !fits(i, 134217727, 512));
      assert(!fits(i, kForm[i].bm * (kTiles + 1), 1));
    }
  const int tests[][3] = {{200, 192, 3},     {200, 192, 512},   {301, 720, 509},  {702, 160, 511},   {702, 4112, 397},
                          {702, 8208, 197}, {2102, 304, 509}, {4102, 1040, 510}, {14402, 4112, 400}, {97, 8208, 5}, {97, 8208, 200}};
  for (auto &t : tests) seen[pick(t[0], t[1], t[2], 256)]++;
  for (int n : seen) assert(n == 1);
}
''')
    exe = str(tmp_path / "f")
    subprocess.check_call(["g++", "-O1", "-std=c++17", "-fsanitize=undefined,address", "-I" + CSRC, str(src), "-o", exe])
    subprocess.check_call([exe], timeout=60)


def fails(xe, call, *args):
    assert call(None, *args) == -1
    return xe.last_error()


def test_valid_arguments_reach_the_ctx(xe, kv, rows):
    L = xe.lib()
    assert fails(xe, L.xe_paged_append_dev, kv, rows) == "null ctx"
    assert fails(xe, L.xe_paged_attn_dev, kv, 0x4000, 0, 0x5000, 4, 1.0, 0, 0x6000, 0) == "null ctx"


@pytest.mark.parametrize("field,value", [
    ("k", None), ("v", None), ("table", None), ("k", 0x1008), ("v", 0x2002), ("hd", 96), ("hd", 0), ("page_size", 8),
    ("page_size", 24), ("page_size", 2048), ("page_size", -16), ("hkv", 0), ("hkv", 1025), ("n_pages", 0), ("batch", 0),
    ("batch", 4097), ("max_pages", 0), ("max_pages", 1 << 27), ("page_stride", 2 * 16 * 64 - 8),
    ("page_stride", 2 * 16 * 64 + 4), ("page_stride", 1 << 62)])
def test_bad_caches_are_refused(xe, kv, rows, field, value):
    setattr(kv, field, value)
    L = xe.lib()
    assert fails(xe, L.xe_paged_append_dev, kv, rows).startswith("paged cache")
    assert fails(xe, L.xe_paged_attn_dev, kv, 0x4000, 0, 0x5000, 4, 1.0, 0, 0x6000, 0).startswith("paged cache")


@pytest.mark.parametrize("change", [
    dict(k=None), dict(v=None), dict(pos=None), dict(n_rows=0), dict(n_rows=4), dict(n_rows=-3), dict(ldkv=127),
    dict(ldkv=1 << 40), dict(ldq=255), dict(ldqo=0), dict(q_out=None), dict(q_out=0x4000, ldqo=512), dict(hq=0),
    dict(hq=1025), dict(q=None), dict(rope_cos=0x9000, rope_len=8), dict(rope_sin=0x9000),
    dict(rope_cos=0x9000, rope_sin=0xa000, rope_len=0), dict(k_norm_w=0x9000, eps=-1.0)])
def test_bad_rows_are_refused(xe, kv, rows, change):
    for f, v in change.items():
        setattr(rows, f, v)
    assert fails(xe, xe.lib().xe_paged_append_dev, kv, rows).startswith("paged append")


@pytest.mark.parametrize("at,value", [(1, None), (3, None), (7, None), (4, 3), (4, 0), (4, 2048), (5, float("inf")),
                                      (5, float("nan")), (6, -1), (2, 255), (8, 255), (2, 1 << 40)])
def test_bad_attention_calls_are_refused(xe, kv, at, value):
    args = [kv, 0x4000, 256, 0x5000, 4, 1.0, 0, 0x6000, 256]
    args[at] = value
    assert fails(xe, xe.lib().xe_paged_attn_dev, *args) not in ("", "null ctx")
    assert xe.lib().xe_paged_attn_dev(None, None, 0x4000, 0, 0x5000, 4, 1.0, 0, 0x6000, 0) == -1


def test_bad_int8_rows_are_refused(xe):
    L = xe.lib()
    good = dict(batch=1, x=0x1000, y=0x2000)
    assert L.xe_w8a8_rows_dev(None, None, xe.W8a8Rows(**good)) == -1 and xe.last_error() == "null ctx or weight"
    for change in (dict(batch=0), dict(batch=513), dict(x=None), dict(y=None), dict(act=-1), dict(act=5),
                   dict(post_w=0x3000), dict(post_w=0x3000, add=0x4000, post_eps=-1.0)):
        assert L.xe_w8a8_rows_dev(None, None, xe.W8a8Rows(**{**good, **change})) == -1
        assert xe.last_error() not in ("", "null ctx or weight"), change
    assert L.xe_w8a8_rows_dev(None, None, None) == -1


def test_structs_match_the_header(xe, tmp_path):
    """Field offsets of the ctypes mirrors are the compiler's."""
    if shutil.which("gcc") is None:
        pytest.skip("no gcc")
    mirrors = {"xe_paged_kv": xe.PagedKV, "xe_paged_rows": xe.PagedRows, "xe_w8a8_rows": xe.W8a8Rows}
    body = "".join('printf("%%zu\\n", sizeof(%s));' % n + "".join('printf("%%zu\\n", offsetof(%s, %s));' % (n, f) for f, _ in c._fields_)
                   for n, c in mirrors.items())
    src = tmp_path / "o.c"
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "xdna_engine.h"\nint main(void) {%s return 0;}' % body)
    exe = str(tmp_path / "o")
    subprocess.check_call(["gcc", "-std=c99", "-I" + os.path.join(ROOT, "include"), str(src), "-o", exe])
    got = [int(x) for x in subprocess.check_output([exe]).split()]
    want = []
    for c in mirrors.values():
        want += [C.sizeof(c)] + [getattr(c, f).offset for f, _ in c._fields_]
    assert got == want
