"""Decoder layers made of the paged cache's operators and the int8 rows, step
after step over caches that fill up.  Every operator's result is checked against
its definition in 64 bits, with what the device held before it as its input: a
code that falls to the other side of a rounding moves no tolerance."""
import numpy as np
import pytest

import oracle_lib as O
from paged_util import EPS16, EPS32, Cache, attn64, f64, heads64, put, rows64, within
from test_rows_q8_gpu import make_weight

pytestmark = pytest.mark.gpu


class Layer:
    """h -> h, with the residual in the epilogues or (post) in the prologues, as
    models with norms behind their sublayers have it."""

    def __init__(self, xe, gpu, rng, batch, d, ffn, hq, hkv, hd, page, max_pages, window, post):
        self.xe, (self.dev, self.ctx) = xe, gpu
        self.dims, self.window, self.post = (batch, d, ffn, hq, hkv, hd), window, post
        n = (hq + 2 * hkv) * hd
        self.w = {name: make_weight(xe, self.ctx, rng, m, k, bias, norm)
                  for name, m, k, bias, norm in (("qkv", n, d, True, 2), ("o", d, hq * hd, False, 0), ("gu", 2 * ffn, d, False, 3),
                                                 ("down", d, ffn, True, 0))}
        self.cache = Cache(xe, self.dev, rng, batch, max_pages, page, hkv, hd)
        self.kv = self.cache.upload()
        self.norm_w = [(0.2 * rng.standard_normal(hd)).astype(np.float32) for _ in range(2)]
        self.post_w = [(0.2 * rng.standard_normal(d)).astype(np.float32) for _ in range(2)]
        self.rope_len = max_pages * page
        at = np.arange(self.rope_len)[:, None] * 1e4 ** (-np.arange(hd // 2) / (hd / 2.0))
        self.rope = np.cos(at).astype(np.float32), np.sin(at).astype(np.float32)
        self.own = [put(xe, self.dev, a) for a in (*self.norm_w, *self.rope, *self.post_w)]

    def free(self):
        self.cache.free()
        for b in self.own:
            b.free()
        for w, _ in self.w.values():
            w.free()

    def rows(self, rec, name, n, x, y, act=0, add=None, post_w=None, total=None, res=None):
        """One linear; rec gets what it read and wrote."""
        xe, (w, defs) = self.xe, self.w[name]
        m, k = defs[0].shape
        outs = m // 2 if act == xe.XE_ACT_GEGLU else m
        self.ctx.synchronize()
        had = [b.read(np.float32, n * c).reshape(n, c) if b else None for b, c in ((x, k), (add, k), (res, outs))]
        p = lambda b: b.ptr if b else None  # noqa: E731
        self.ctx.w8a8_rows_dev(w, xe.W8a8Rows(n, x.ptr, y.ptr, act=act, add=p(add), post_w=p(post_w[0]) if post_w else None,
                                              sum=p(total), res=p(res)))
        rec.append((name, defs, had, post_w[1] if post_w else None, act, y, outs, total, k, n))

    def check_rows(self, rec):
        for name, defs, (x, add, res), post, act, y, outs, total, k, n in rec:
            want, t, bound = rows64(*defs, x, add, post, act, res)
            if total is not None:
                within(total.read(np.float32, n * k).reshape(n, k), t.astype(np.float64), 2 ** -23 * np.abs(t) + 1e-30, name)
            within(y.read(np.float32, n * outs).reshape(n, outs), want, bound, name)
        rec.clear()

    def append(self, bufs, n, pos, counts):
        """Appends n rows of bufs["qkv"]; the host's cache follows the device's,
        whose new rows are checked."""
        xe, c = self.xe, self.cache
        _, _, _, hq, hkv, hd = self.dims
        ld, base = (hq + 2 * hkv) * hd, bufs["qkv"].ptr
        qn, kn, cos, sin = (b.ptr for b in self.own[:4])
        self.ctx.paged_append_dev(self.kv, xe.PagedRows(
            n, hq, q=base, k=base + 4 * hq * hd, v=base + 4 * (hq + hkv) * hd, ldq=ld, ldkv=ld, q_out=bufs["q"].ptr, ldqo=hq * hd,
            pos=bufs["pos"].ptr, start=bufs["start"].ptr if counts is not None else None, q_norm=qn, k_norm=kn, cos=cos, sin=sin,
            rope_len=self.rope_len))
        self.ctx.synchronize()
        x = bufs["qkv"].read(np.float32, n * ld).reshape(n, ld)
        gq = bufs["q"].read(np.float32, n * hq * hd).reshape(n, hq, hd)
        gk, gv = c.read()
        page, i = c.dims[2], 0
        for b, cnt in enumerate(counts if counts is not None else [1] * n):
            for j in range(cnt):
                at = int(pos[b]) + j
                row, i = i, i + 1
                if pos[b] < 0:
                    continue
                q, k, v = np.split(x[row].reshape(-1, hd), [hq, hq + hkv])
                pg = c.table[b, at // page]
                for g in range(hkv):
                    o = (g * page + at % page) * hd
                    c.v[pg, o:o + hd] = O.bf16_bits(v[g])
                    want = heads64(k[g:g + 1], self.norm_w[1], 1e-6, *self.rope, at)[0]
                    big = np.abs(np.roll(want, hd // 2)) + np.abs(want)
                    got = gk[pg, o:o + hd]
                    within(f64(got), want, EPS16 * np.abs(want) + (hd / 2 + 16) * EPS32 * big, "k")
                    c.k[pg, o:o + hd] = got
                want = heads64(q, self.norm_w[0], 1e-6, *self.rope, at)
                within(gq[row], want, (hd / 2 + 16) * EPS32 * (np.abs(np.roll(want, hd // 2, 1)) + np.abs(want)), "q")
        assert np.array_equal(gk, c.k) and np.array_equal(gv, c.v), "only the new rows change"
        return gq

    def step(self, bufs, pos):
        """One token of every stream with pos >= 0."""
        batch, d, ffn, hq, hkv, hd = self.dims
        rec = []
        self.rows(rec, "qkv", batch, bufs["h"], bufs["qkv"])
        self.ctx.synchronize()
        self.check_rows(rec)
        gq = self.append(bufs, batch, pos, None)
        lens = np.maximum(pos + 1, 0)
        bufs["lens"].write(lens.astype(np.int32))
        self.ctx.paged_attn_dev(self.kv, bufs["q"], bufs["lens"], hq, hd ** -0.5, bufs["o"], window=self.window)
        self.ctx.synchronize()
        want, bound = attn64(self.cache, gq, lens, hq, hd ** -0.5, self.window)
        within(bufs["o"].read(np.float32, batch * hq * hd).reshape(batch, hq, hd), want, bound, "attention")
        gelu = self.xe.XE_ACT_GEGLU
        if self.post:
            self.rows(rec, "o", batch, bufs["o"], bufs["t"])
            self.rows(rec, "gu", batch, bufs["h"], bufs["f"], act=gelu, add=bufs["t"], post_w=(self.own[4], self.post_w[0]),
                      total=bufs["h2"])
            self.rows(rec, "down", batch, bufs["f"], bufs["h"], res=bufs["h2"])
        else:
            self.rows(rec, "o", batch, bufs["o"], bufs["h2"], res=bufs["h"])
            self.rows(rec, "gu", batch, bufs["h2"], bufs["f"], act=gelu)
            self.rows(rec, "down", batch, bufs["f"], bufs["h"], res=bufs["h2"])
        self.ctx.synchronize()
        self.check_rows(rec)


@pytest.mark.parametrize("batch,d,ffn,hq,hkv,hd,page", [(1, 256, 512, 4, 1, 64, 16), (5, 384, 400, 6, 2, 128, 32), (20, 256, 320, 4, 1, 256, 16),
                                                        (70, 128, 192, 8, 8, 64, 16)])
def test_layers_step_by_step(gpu, xe, batch, d, ffn, hq, hkv, hd, page):
    """A prompt, then single tokens across the ends of pages; two layers, one with
    a window and norms behind its sublayers; every third stream idle at times."""
    dev, ctx = gpu
    print("[case] layers batch %d d %d heads %d/%d x %d" % (batch, d, hq, hkv, hd), flush=True)
    rng = np.random.default_rng(batch + d)
    layers = [Layer(xe, gpu, rng, batch, d, ffn, hq, hkv, hd, page, 5, window, post) for window, post in ((0, False), (page + 3, True))]
    counts = rng.integers(0, 2 * page, batch)
    counts[0] = page - 2  # the third new token begins a page
    ld, n = (hq + 2 * hkv) * hd, max(int(counts.sum()), batch)
    bufs = {name: xe.Buf(dev, max(s, 1) * 4) for name, s in (
        ("h", batch * d), ("h2", batch * d), ("t", batch * d), ("qkv", n * ld), ("q", n * hq * hd), ("o", batch * hq * hd),
        ("f", batch * ffn), ("pos", batch), ("start", batch + 1), ("lens", batch))}
    pos = np.zeros(batch, np.int32)
    for layer in layers:
        bufs["pos"].write(pos)
        bufs["start"].write(np.concatenate([[0], np.cumsum(counts)]).astype(np.int32))
        bufs["qkv"].write(rng.standard_normal((n, ld)).astype(np.float32))
        layer.append(bufs, int(counts.sum()), pos, counts)
    pos = counts.astype(np.int32)
    for step in range(5):
        now = pos.copy()
        now[2::3] = np.where(step % 2, -1, now[2::3])
        bufs["pos"].write(now)
        bufs["h"].write(rng.standard_normal((batch, d)).astype(np.float32))
        for layer in layers:
            layer.step(bufs, now)
        pos += now >= 0
    for x in (*layers, *bufs.values()):
        x.free()


def test_two_contexts(gpu, xe):
    """Calls of two contexts of one device in turn, without a wait between them:
    each has its workspace, and the results are those of one alone."""
    dev, ctx = gpu
    other = xe.CtxDecode(dev)
    rng = np.random.default_rng(3)
    c = Cache(xe, dev, rng, 3, 60, 16, 2, 128)
    kv = c.upload()
    q = rng.standard_normal((3, 8 * 128)).astype(np.float32)
    x = rng.standard_normal((100, 512)).astype(np.float32)
    bq, bl, bx = put(xe, dev, q), put(xe, dev, np.array([960, 7, 500], np.int32)), put(xe, dev, x)
    both = []
    for one in (ctx, other):
        w, _ = make_weight(xe, one, np.random.default_rng(4), 300, 512, True, 2)
        both.append((one, w, [xe.Buf(dev, q.nbytes) for _ in range(6)], [xe.Buf(dev, 100 * 300 * 4) for _ in range(6)]))
    for i in range(6):
        for one, w, outs, ys in both:
            one.paged_attn_dev(kv, bq, bl, 8, 0.1, outs[i])
            one.w8a8_rows_dev(w, xe.W8a8Rows(100, bx.ptr, ys[i].ptr))
    for one, *_ in both:
        one.synchronize()
    for pick, size in ((2, q.size), (3, 100 * 300)):
        got = [b.read(np.uint32, size) for t in both for b in t[pick]]
        assert all(np.array_equal(got[0], g) for g in got)
    want, bound = attn64(c, q.reshape(3, 8, 128), [960, 7, 500], 8, 0.1)
    within(both[0][2][0].read(np.float32, q.size).reshape(3, 8, 128), want, bound, "attention")
    for _, w, outs, ys in both:
        w.free()
        for b in (*outs, *ys):
            b.free()
    for b in (bq, bl, bx, c):
        b.free()
    other.close()
