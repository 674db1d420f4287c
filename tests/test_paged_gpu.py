"""Paged KV cache on the GPU: appended rows bit for bit where they are only
rounded, everything else against 64 bits within derived bounds; lengths of
zero and one, pages that end inside a tile, missing pages, poisoned slots,
strides, windows, and the order of calls."""
import math

import numpy as np
import pytest

import oracle_lib as O
from paged_util import EPS16, EPS32, At, Cache, attn64, f64, heads64, put, within

pytestmark = pytest.mark.gpu

HEADS = [(12, 12, 64), (4, 1, 256), (8, 2, 128), (6, 2, 64), (7, 1, 128), (40, 2, 64), (16, 1, 256), (24, 1, 128)]


def rope_table(n, hd):
    at = np.arange(n)[:, None] * 1e6 ** (-np.arange(hd // 2) / (hd / 2.0))
    return np.cos(at).astype(np.float32), np.sin(at).astype(np.float32)


def append_case(xe, gpu, seed, hq, hkv, hd, page, counts, pos, norm, rope, gap=0, pad=0, off=0, behind=0, spoil=None,
                decode=False, with_q=True):
    """One append; checks every byte of the pool and of q_out."""
    dev, ctx = gpu
    rng = np.random.default_rng(seed)
    batch = len(counts)
    max_pages = -(-max(max(p + c for p, c in zip(pos, counts)), 1) // page)
    c = Cache(xe, dev, rng, batch, max_pages, page, hkv, hd, gap=gap)
    if spoil is not None:
        spoil(c)
    kv = c.upload()
    start = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
    n = int(start[-1]) + behind
    ld = (hq + 2 * hkv) * hd + pad
    x = rng.standard_normal((n, ld)).astype(np.float32)
    flat = np.concatenate([np.zeros(off, np.float32), x.reshape(-1)])
    w = [0.2 * rng.standard_normal(hd).astype(np.float32) for _ in range(2)] if norm else [None, None]
    cos, sin = rope_table(max_pages * page, hd) if rope else (None, None)
    bufs = {"x": put(xe, dev, flat), "pos": put(xe, dev, np.array(pos, np.int32)), "start": put(xe, dev, start)}
    for name, a in (("qn", w[0]), ("kn", w[1]), ("cos", cos), ("sin", sin)):
        if a is not None:
            bufs[name] = put(xe, dev, a)
    ldqo = hq * hd + pad
    mark = np.full(n * ldqo + off, 7.5, np.float32)
    bufs["q_out"] = put(xe, dev, mark)
    base = bufs["x"].ptr + 4 * off
    p = lambda name: bufs[name].ptr if name in bufs else None  # noqa: E731
    rows = xe.PagedRows(n, hq, q=base if with_q else None, k=base + 4 * hq * hd, v=base + 4 * (hq + hkv) * hd,
                        ldq=ld, ldkv=ld, q_out=p("q_out") + 4 * off if with_q else None, ldqo=ldqo, pos=p("pos"),
                        start=None if decode else p("start"), q_norm=p("qn") if with_q else None, k_norm=p("kn"), eps=1e-6,
                        cos=p("cos"), sin=p("sin"), rope_len=max_pages * page if rope else 0)
    ctx.paged_append_dev(kv, rows)
    ctx.synchronize()
    gk, gv = c.read()
    got_q = bufs["q_out"].read(np.float32, mark.size)[off:].reshape(n, ldqo)
    want_k, want_v, left = c.k.copy(), c.v.copy(), np.ones(c.k.shape, bool)
    q_left = np.ones(got_q.shape, bool)
    for b in range(batch):
        for i in range(int(start[b]), int(start[b + 1])):
            at = pos[b] + i - int(start[b])
            if pos[b] < 0 or at >= max_pages * page or not 0 <= c.table[b, at // page] < c.n_pages:
                continue
            pg = c.table[b, at // page]
            q, k, v = np.split(x[i, :(hq + 2 * hkv) * hd].reshape(-1, hd), [hq, hq + hkv])
            for g in range(hkv):
                o = (g * page + at % page) * hd
                left[pg, o:o + hd] = False
                assert np.array_equal(gv[pg, o:o + hd], O.bf16_bits(v[g])), "values are rounded to nearest, ties to even"
                if not norm and not rope:
                    assert np.array_equal(gk[pg, o:o + hd], O.bf16_bits(k[g]))
                want = heads64(k[g:g + 1], w[1], 1e-6, cos, sin, at)[0]
                big = np.abs(np.concatenate([want[hd // 2:], want[:hd // 2]])) + np.abs(want)
                within(f64(gk[pg, o:o + hd]), want, EPS16 * np.abs(want) + (hd / 2 + 16) * EPS32 * big, "k")
            if with_q:
                q_left[i, :hq * hd] = False
                want = heads64(q, w[0], 1e-6, cos, sin, at)
                big = np.abs(np.roll(want, hd // 2, 1)) + np.abs(want)
                within(got_q[i, :hq * hd].reshape(hq, hd), want, (hd / 2 + 16) * EPS32 * big, "q")
    assert np.array_equal(gk[left], want_k[left]) and np.array_equal(gv[left], want_v[left]), "other slots stay"
    assert np.all(got_q[q_left] == 7.5), "rows left out stay"
    c.free()
    for b in bufs.values():
        b.free()


@pytest.mark.parametrize("hq,hkv,hd", HEADS)
@pytest.mark.parametrize("norm,rope", [(False, False), (True, True), (False, True), (True, False)])
def test_append_prompts(gpu, xe, hq, hkv, hd, norm, rope):
    print("[case] append %d/%d x %d norm %d rope %d" % (hq, hkv, hd, norm, rope), flush=True)
    append_case(xe, gpu, hd + hq, hq, hkv, hd, 16, [5, 0, 1, 33, 0, 16, 0], [0, 3, 31, 7, 0, 16, 2], norm, rope)


@pytest.mark.parametrize("page", [16, 64, 1024])
def test_append_one_row_a_stream(gpu, xe, page):
    append_case(xe, gpu, page, 4, 1, 256, page, [1] * 70, [(37 * b) % 200 for b in range(70)], True, True, decode=True)


def test_append_one_row(gpu, xe):
    append_case(xe, gpu, 1, 4, 1, 256, 16, [1], [0], True, True, decode=True)
    append_case(xe, gpu, 2, 12, 12, 64, 16, [1], [15], False, False, decode=True)


@pytest.mark.parametrize("pad,off", [(4, 0), (1, 0), (0, 1), (3, 2)])
def test_append_strides_and_alignment(gpu, xe, pad, off):
    """Row strides that are no multiple of 16 bytes, rows that start off one."""
    append_case(xe, gpu, 10 * pad + off, 8, 2, 128, 32, [3, 9], [30, 0], True, True, pad=pad, off=off)


def test_append_interleaved_pool(gpu, xe):
    append_case(xe, gpu, 5, 8, 2, 128, 16, [3, 20], [14, 1], False, True, gap=264)


def test_append_without_queries(gpu, xe):
    append_case(xe, gpu, 6, 8, 2, 128, 16, [3, 20], [14, 1], True, True, with_q=False)


def test_append_leaves_rows_out(gpu, xe):
    """Rows behind the last stream, streams at a negative position, missing and
    impossible pages: nothing of them is written."""
    def spoil(c):
        c.table[1, 1] = -1
        c.table[3, 0] = c.n_pages
        c.table[3, 1] = 2 ** 31 - 1
    append_case(xe, gpu, 7, 4, 2, 64, 16, [4, 30, 5, 20, 2], [0, 10, -3, 0, 8], True, True, behind=9, spoil=spoil)


def test_append_past_table_and_rope(gpu, xe):
    """Positions past the table, or past the rotation's rows: left out."""
    dev, ctx = gpu
    rng = np.random.default_rng(3)
    c = Cache(xe, dev, rng, 3, 2, 16, 1, 64)
    kv = c.upload()
    x, cos, sin = rng.standard_normal((3, 128)).astype(np.float32), *rope_table(20, 64)
    bufs = [put(xe, dev, a) for a in (x, np.array([32, 20, 2 ** 31 - 1], np.int32), cos, sin)]
    rows = xe.PagedRows(3, 0, k=bufs[0].ptr, v=bufs[0].ptr + 256, ldkv=128, pos=bufs[1].ptr, cos=bufs[2].ptr,
                        sin=bufs[3].ptr, rope_len=20)
    ctx.paged_append_dev(kv, rows)
    ctx.synchronize()
    k, v = c.read()
    assert np.array_equal(k, c.k) and np.array_equal(v, c.v)
    c.free()
    for b in bufs:
        b.free()


def test_append_in_place_queries(gpu, xe):
    """q_out over q gives what a q_out of its own gives."""
    dev, ctx = gpu
    rng = np.random.default_rng(4)
    c = Cache(xe, dev, rng, 5, 4, 16, 2, 128)
    kv = c.upload()
    x = rng.standard_normal((5, 8 * 128)).astype(np.float32)
    cos, sin = rope_table(64, 128)
    bx, bo, bp, bc, bs = (put(xe, dev, a) for a in (x, np.zeros((5, 512), np.float32), np.arange(5, dtype=np.int32) * 13, cos, sin))
    kw = dict(q=bx.ptr, k=bx.ptr + 4 * 512, v=bx.ptr + 4 * 768, ldq=1024, ldkv=1024, pos=bp.ptr, cos=bc.ptr, sin=bs.ptr, rope_len=64)
    ctx.paged_append_dev(kv, xe.PagedRows(5, 4, q_out=bo.ptr, ldqo=512, **kw))
    ctx.paged_append_dev(kv, xe.PagedRows(5, 4, q_out=bx.ptr, ldqo=1024, **kw))
    ctx.synchronize()
    a, b = bo.read(np.float32, 5 * 512).reshape(5, 512), bx.read(np.float32, 5 * 1024).reshape(5, 1024)
    assert np.array_equal(a, b[:, :512]) and np.array_equal(b[:, 512:], x[:, 512:])
    c.free()
    for t in (bx, bo, bp, bc, bs):
        t.free()


# ---------------------------------------------------------------------------

def attn_case(xe, gpu, seed, hq, hkv, hd, page, lens, max_pages, window=0, gap=0, change=None, poison=True, scale=None, pad=0,
              rel=1e-5):
    """One attention call, twice, against 64 bits; slots that no stream may
    read hold NaN."""
    dev, ctx = gpu
    rng = np.random.default_rng(seed)
    batch = len(lens)
    c = Cache(xe, dev, rng, batch, max_pages, page, hkv, hd, gap=gap)
    if change is not None:
        change(c)
    if poison:
        used = np.zeros((c.n_pages, page), bool)
        for b in range(batch):
            n = min(max(int(lens[b]), 0), max_pages * page)
            for t in range(max(0, int(lens[b]) - window) if window else 0, n):
                if 0 <= c.table[b, t // page] < c.n_pages:
                    used[c.table[b, t // page], t % page] = True
        for bits in (c.k, c.v):
            body = bits[:, :c.dense].reshape(c.n_pages, hkv, page, hd)
            body.transpose(0, 2, 1, 3)[~used] = 0x7FC0
            bits[:, c.dense:] = 0x7F80
    kv = c.upload()
    q = rng.standard_normal((batch, hq, hd)).astype(np.float32)
    wide = np.full((batch, hq * hd + pad), np.nan, np.float32)
    wide[:, :hq * hd] = q.reshape(batch, -1)
    scale = 1.0 / math.sqrt(hd) if scale is None else scale
    bufs = [put(xe, dev, wide), put(xe, dev, np.array(lens, np.int32)),
            put(xe, dev, np.full((batch, hq * hd + pad), 3.25, np.float32))]
    ld = hq * hd + pad if pad else 0
    got = []
    for _ in range(2):
        ctx.paged_attn_dev(kv, bufs[0], bufs[1], hq, scale, bufs[2], window=window, ldq=ld, ldo=ld)
        ctx.synchronize()
        got.append(bufs[2].read(np.float32, wide.size).reshape(batch, -1))
    assert np.array_equal(got[0].view(np.uint32), got[1].view(np.uint32)), "the same call gives the same bits"
    assert np.all(got[0][:, hq * hd:] == 3.25)
    out = got[0][:, :hq * hd].reshape(batch, hq, hd)
    want, bound = attn64(c, q, lens, hq, scale, window)
    within(out, want, bound, "attention")
    norm = np.linalg.norm(want)
    assert np.linalg.norm(out - want) <= rel * norm
    empty = ~np.any(want != 0, axis=(1, 2))
    assert np.all(out[empty] == 0)
    c.free()
    for b in bufs:
        b.free()
    return out


@pytest.mark.parametrize("hq,hkv,hd", HEADS)
@pytest.mark.parametrize("page", [16, 64])
def test_attn_lengths(gpu, xe, hq, hkv, hd, page):
    print("[case] paged attention %d/%d x %d page %d" % (hq, hkv, hd, page), flush=True)
    attn_case(xe, gpu, hq + hd + page, hq, hkv, hd, page, [1, 0, 15, 16, 17, 63, 64, 65, 200, 384], 384 // page)


@pytest.mark.parametrize("hq,hkv,hd", [(12, 12, 64), (4, 1, 256), (16, 2, 128)])
@pytest.mark.parametrize("n", [1, 2, 31, 33, 1000, 4096, 5003])
def test_attn_one_stream(gpu, xe, hq, hkv, hd, n):
    print("[case] one stream %d/%d x %d, %d keys" % (hq, hkv, hd, n), flush=True)
    attn_case(xe, gpu, n + hd, hq, hkv, hd, 32, [n], -(-n // 32) + 2)


@pytest.mark.parametrize("window", [1, 5, 16, 64, 100, 1000])
def test_attn_window(gpu, xe, window):
    attn_case(xe, gpu, window, 4, 1, 256, 16, [1, 0, window - 1, window, window + 1, 300, 416], 26, window=window)
    attn_case(xe, gpu, window, 12, 12, 64, 32, [1, 300, 416], 13, window=window)


def test_attn_missing_pages(gpu, xe):
    """Pages that a stream has not: at its start, in its middle, all of them;
    entries far out of the pool."""
    def change(c):
        c.table[0, :5] = -1
        c.table[1, 7] = c.n_pages
        c.table[1, 9] = 2 ** 31 - 1
        c.table[2, :] = -2 ** 31
        c.table[3, 11] = -1
    attn_case(xe, gpu, 9, 8, 2, 128, 16, [180, 192, 150, 177], 12, change=change)
    attn_case(xe, gpu, 9, 8, 2, 128, 16, [180, 192, 150, 177], 12, change=change, window=30)


def test_attn_lengths_outside_the_table(gpu, xe):
    attn_case(xe, gpu, 11, 4, 2, 64, 16, [-1, -2 ** 31, 2 ** 31 - 1, 65, 64, 100], 4)
    attn_case(xe, gpu, 11, 4, 2, 64, 16, [-1, -2 ** 31, 2 ** 31 - 1, 65, 64, 100], 4, window=50)


def test_attn_interleaved_pool_and_strides(gpu, xe):
    attn_case(xe, gpu, 12, 8, 2, 128, 16, [33, 100, 7], 7, gap=1032)
    attn_case(xe, gpu, 13, 7, 1, 64, 16, [33, 100, 7], 7, pad=3)


@pytest.mark.parametrize("batch", [65, 130, 600])
def test_attn_many_streams(gpu, xe, batch):
    rng = np.random.default_rng(batch)
    lens = rng.integers(0, 97, batch)
    lens[::7] = 0
    lens[batch // 2] = 96
    attn_case(xe, gpu, batch, 2, 1, 64, 16, lens, 6)


def test_attn_most_streams(gpu, xe):
    rng = np.random.default_rng(4096)
    attn_case(xe, gpu, 24, 2, 1, 64, 16, rng.choice([0, 1, 16, 17, 32], 4096), 2)


@pytest.mark.parametrize("hq,hkv,batch", [(1024, 1, 2), (1024, 1, 70), (1024, 1024, 3), (48, 16, 2), (48, 16, 70)])
def test_attn_many_heads(gpu, xe, hq, hkv, batch):
    attn_case(xe, gpu, hq + hkv, hq, hkv, 64, 16, [18, 3] * (batch // 2) + [0] * (batch % 2), 2)


@pytest.mark.parametrize("hq,hkv,hd", [(2, 1, 64), (20, 1, 128)])
def test_attn_one_long_stream_among_short_ones(gpu, xe, hq, hkv, hd):
    """Its partials meet on three levels; the others read its first page."""
    dev, ctx = gpu
    print("[case] one stream of 60001 keys among 65, %d/%d x %d" % (hq, hkv, hd), flush=True)
    rng = np.random.default_rng(25)
    page, n, batch = 256, 60001, 65
    c = Cache(xe, dev, rng, 1, -(-n // page), page, hkv, hd)
    table = np.full((batch, c.table.shape[1]), -1, np.int32)
    table[30] = c.table[0]
    table[:, 0] = c.table[0, 0]
    c.table, c.dims = table, (batch,) + c.dims[1:]
    lens = np.arange(batch, dtype=np.int32) % 17
    lens[30] = n
    q = rng.standard_normal((batch, hq, hd)).astype(np.float32)
    kv = c.upload()
    bufs = [put(xe, dev, a) for a in (q, lens, np.full(q.shape, 3.25, np.float32))]
    want, bound = attn64(c, q, lens, hq, hd ** -0.5)
    for _ in range(3):
        ctx.paged_attn_dev(kv, bufs[0], bufs[1], hq, hd ** -0.5, bufs[2])
        ctx.synchronize()
        within(bufs[2].read(np.float32, q.size).reshape(q.shape), want, bound, "attention")
    c.free()
    for b in bufs:
        b.free()


@pytest.mark.parametrize("hq,hkv,hd,lens", [(4, 1, 256, [3000, 0, 17]), (20, 1, 128, [700]), (2, 1, 64, list(range(0, 700, 10)))])
def test_attn_over_its_queries(gpu, xe, hq, hkv, hd, lens):
    dev, ctx = gpu
    rng = np.random.default_rng(len(lens))
    c = Cache(xe, dev, rng, len(lens), -(-max(lens) // 16), 16, hkv, hd)
    kv = c.upload()
    q = rng.standard_normal((len(lens), hq, hd)).astype(np.float32)
    bufs = [put(xe, dev, a) for a in (q, np.array(lens, np.int32), q)]
    ctx.paged_attn_dev(kv, bufs[0], bufs[1], hq, 0.1, bufs[0])
    ctx.paged_attn_dev(kv, bufs[2], bufs[1], hq, 0.1, bufs[2])
    ctx.synchronize()
    want, bound = attn64(c, q, lens, hq, 0.1)
    for b in (bufs[0], bufs[2]):
        within(b.read(np.float32, q.size).reshape(q.shape), want, bound, "over the queries")
    c.free()
    for b in bufs:
        b.free()


def test_attn_all_idle(gpu, xe):
    attn_case(xe, gpu, 14, 4, 1, 256, 16, [0, 0, 0], 2)


def test_attn_large_scores(gpu, xe):
    """Scores of some hundreds: the softmax is one key's weight, no overflow."""
    attn_case(xe, gpu, 15, 4, 1, 256, 16, [200, 33], 13, scale=40.0, rel=2e-3)
    attn_case(xe, gpu, 16, 4, 1, 256, 16, [200, 33], 13, scale=-3.0, rel=2e-4)
    attn_case(xe, gpu, 17, 4, 1, 256, 16, [200, 33], 13, scale=0.0)


def test_attn_shared_prefix(gpu, xe):
    """Streams that share their first pages."""
    def change(c):
        c.table[1:, :3] = c.table[0, :3]
    attn_case(xe, gpu, 18, 8, 2, 128, 16, [100, 49, 48, 60], 7, change=change)


def test_attn_infinite_value(gpu, xe):
    """An infinity among the values: no number or infinite in that dimension, the
    others untouched by it."""
    dev, ctx = gpu
    rng = np.random.default_rng(19)
    for n in (40, 3000):
        c = Cache(xe, dev, rng, 1, -(-n // 16), 16, 1, 64)
        q = rng.standard_normal((1, 4, 64)).astype(np.float32)
        want, bound = attn64(c, q, [n], 4, 0.125)
        for t in (3, n - 1):
            c.slot(c.v, c.table[0, t // 16], 0, t % 16)[5] = 0x7F80
        kv = c.upload()
        bufs = [put(xe, dev, a) for a in (q, np.array([n], np.int32), np.zeros_like(q))]
        ctx.paged_attn_dev(kv, bufs[0], bufs[1], 4, 0.125, bufs[2])
        ctx.synchronize()
        out = bufs[2].read(np.float32, q.size).reshape(1, 4, 64)
        assert not np.any(np.isfinite(out[..., 5]))
        keep = np.arange(64) != 5
        within(out[..., keep], want[..., keep], bound, "beside infinity")
        c.free()
        for b in bufs:
            b.free()


def test_attn_changing_calls(gpu, xe):
    """Calls of other sizes in between leave a call's result as it was."""
    first = attn_case(xe, gpu, 20, 4, 1, 256, 16, [700, 3, 90], 44)
    attn_case(xe, gpu, 21, 12, 12, 64, 32, [1500], 47)
    attn_case(xe, gpu, 22, 16, 2, 128, 16, [5] * 40, 1)
    assert np.array_equal(first, attn_case(xe, gpu, 20, 4, 1, 256, 16, [700, 3, 90], 44))


def test_far_pages(gpu, xe):
    """Pages whose elements lie beyond 2^32: an interleaved pool with wide gaps."""
    dev, ctx = gpu
    rng = np.random.default_rng(23)
    page, hkv, hd = 16, 1, 64
    stride = (1 << 32) // 7 // 8 * 8
    n_pages = 10  # the last ones start past 2^32 elements
    need = (n_pages - 1) * stride + hkv * page * hd
    bk, bv = xe.Buf(dev, need * 2), xe.Buf(dev, need * 2)
    table = np.array([[9, 0, 8]], np.int32)
    bt = put(xe, dev, table)
    n = 41
    x = rng.standard_normal((n, 3 * hd)).astype(np.float32)
    bx, bp, bs, bq = put(xe, dev, x), put(xe, dev, np.zeros(1, np.int32)), put(xe, dev, np.array([0, n], np.int32)), xe.Buf(dev, n * hd * 4)
    kv = xe.PagedKV(bk, bv, bt, n_pages, hkv, page, hd, 1, 3, page_stride=stride)
    ctx.paged_append_dev(kv, xe.PagedRows(n, 1, q=bx.ptr, k=bx.ptr + 4 * hd, v=bx.ptr + 8 * hd, ldq=3 * hd, ldkv=3 * hd,
                                          q_out=bq.ptr, ldqo=hd, pos=bp.ptr, start=bs.ptr))
    bl, bo = put(xe, dev, np.array([n], np.int32)), xe.Buf(dev, hd * 4)
    ctx.paged_attn_dev(kv, At(bq.ptr + (n - 1) * hd * 4), bl, 1, 0.125, bo)
    ctx.synchronize()
    out = bo.read(np.float32, hd).astype(np.float64)
    k, v = (f64(O.bf16_bits(x[:, a * hd:(a + 1) * hd])) for a in (1, 2))
    s = (k @ x[-1, :hd].astype(np.float64)) * 0.125
    p = np.exp(s - s.max())
    want = (p / p.sum()) @ v
    assert np.linalg.norm(out - want) <= 1e-5 * np.linalg.norm(want)
    for b in (bk, bv, bt, bx, bp, bs, bq, bl, bo):
        b.free()
