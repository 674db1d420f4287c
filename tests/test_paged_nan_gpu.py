"""Queries and keys that are no numbers, in the paged attention: NaN in the
heads that meet them and nowhere else, in whichever form and on whichever level
of merges a stream's keys come together."""
import numpy as np
import pytest

import oracle_lib as O
from paged_util import Cache, attn64, put, within

pytestmark = pytest.mark.gpu

# Streams' lengths: few streams take whole workgroups of eight waves (1 stream of
# up to 512 keys one, of up to 6144 one group of partials, beyond that two
# levels), more than 64 share all keys equally in workgroups of four waves.
FEW = [300, 3000, 9000]


def lens_of(form, n):
    """Stream 1 has n keys."""
    return [40, n, 0, 17] if form == "whole" else [9 * (b % 5) for b in range(30)] + [n] + [40] * 40


def call(xe, gpu, c, q, lens, hq, window=0):
    dev, ctx = gpu
    kv = c.upload()
    bufs = [put(xe, dev, a) for a in (q, np.array(lens, np.int32), np.full(q.shape, 3.25, np.float32))]
    ctx.paged_attn_dev(kv, bufs[0], bufs[1], hq, 0.125, bufs[2], window=window)
    ctx.synchronize()
    out = bufs[2].read(np.float32, q.size).reshape(q.shape)
    c.free()
    for b in bufs:
        b.free()
    return out


def setup(xe, gpu, form, n, hkv, hd, seed):
    rng = np.random.default_rng(seed)
    lens = lens_of(form, n)
    b = lens.index(n)
    c = Cache(xe, gpu[0], rng, 1, -(-n // 64), 64, hkv, hd)
    table = np.full((len(lens), c.table.shape[1]), -1, np.int32)
    table[:, 0] = np.setdiff1d(np.arange(c.n_pages), c.table)[0]  # the short streams' page
    table[b] = c.table[0]
    c.table, c.dims = table, (len(lens),) + c.dims[1:]
    return rng, lens, b, c


@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
@pytest.mark.parametrize("hq,hkv,hd", [(4, 1, 64), (4, 2, 128), (40, 2, 256)])
@pytest.mark.parametrize("n", FEW)
@pytest.mark.parametrize("form", ["whole", "shares"])
def test_query_that_is_no_number(gpu, xe, form, n, hq, hkv, hd, bad):
    print("[case] %s %s, %d keys, %d/%d x %d" % (bad, form, n, hq, hkv, hd), flush=True)
    rng, lens, b, c = setup(xe, gpu, form, n, hkv, hd, n + hd)
    q = rng.standard_normal((len(lens), hq, hd)).astype(np.float32)
    want, bound = attn64(c, q, lens, hq, 0.125)
    spoiled = q.copy()
    spoiled[b, hq - 1, 5] = bad
    idle = lens.index(0)
    spoiled[idle, 0] = bad  # no keys: zeros, whatever the query
    out = call(xe, gpu, c, spoiled, lens, hq)
    assert np.all(np.isnan(out[b, hq - 1]))
    keep = np.ones((len(lens), hq), bool)
    keep[b, hq - 1] = False
    within(out[keep], want[keep], bound[keep], "beside it")
    assert np.all(out[idle] == 0)


@pytest.mark.parametrize("run", ["one", "tile", "share", "many", "last", "all"])
@pytest.mark.parametrize("hq,hkv,hd", [(8, 2, 64), (2, 1, 256)])
@pytest.mark.parametrize("n", FEW)
@pytest.mark.parametrize("form", ["whole", "shares"])
def test_keys_that_are_no_numbers(gpu, xe, form, n, hq, hkv, hd, run):
    """One key, 16, a workgroup's whole share (of 3000 keys: 12 tiles of 16 a
    workgroup), many of them, the newest key, all: NaN in the heads of that kv
    head, the other kv heads and streams untouched."""
    print("[case] %s NaN keys, %s, %d keys, %d/%d x %d" % (run, form, n, hq, hkv, hd), flush=True)
    rng, lens, b, c = setup(xe, gpu, form, n, hkv, hd, n + hd + 1)
    q = rng.standard_normal((len(lens), hq, hd)).astype(np.float32)
    want, bound = attn64(c, q, lens, hq, 0.125)
    first, last = {"one": (200, 201), "tile": (208, 224), "share": (192, min(n, 384)), "many": (64, n - 30),
                   "last": (n - 1, n), "all": (0, n)}[run]
    g = hkv - 1
    for t in range(first, last):
        c.slot(c.k, c.table[b, t // 64], g, t % 64)[t % hd] = 0x7FC0
    out = call(xe, gpu, c, q, lens, hq)
    heads = np.arange(hq) // (hq // hkv) == g
    assert np.all(np.isnan(out[b, heads]))
    keep = np.ones((len(lens), hq), bool)
    keep[b, heads] = False
    within(out[keep], want[keep], bound[keep], "beside them")


@pytest.mark.parametrize("n", FEW)
@pytest.mark.parametrize("form", ["whole", "shares"])
def test_keys_before_the_window(gpu, xe, form, n):
    """Keys, and their values, that are no numbers before the window change nothing."""
    rng, lens, b, c = setup(xe, gpu, form, n, 1, 64, n)
    window = n - 130
    lens = [min(x, window) if x != n else x for x in lens]
    q = rng.standard_normal((len(lens), 4, 64)).astype(np.float32)
    want, bound = attn64(c, q, lens, 4, 0.125, window)
    for t in range(64, 130):
        for bits in (c.k, c.v):
            c.slot(bits, c.table[b, t // 64], 0, t % 64)[:] = 0x7FC0
    out = call(xe, gpu, c, q, lens, 4, window)
    within(out, want, bound, "window")


@pytest.mark.parametrize("n", FEW)
@pytest.mark.parametrize("form", ["whole", "shares"])
@pytest.mark.parametrize("bad", [np.inf, -np.inf])
def test_infinite_key(gpu, xe, form, n, bad):
    """NaN, or, where its score is minus infinity, the result without that key."""
    rng, lens, b, c = setup(xe, gpu, form, n, 1, 64, n + 7)
    q = rng.standard_normal((len(lens), 4, 64)).astype(np.float32)
    t = n - 2
    c.slot(c.k, c.table[b, t // 64], 0, t % 64)[9] = O.bf16_bits(np.array([bad], np.float32))[0]
    out = call(xe, gpu, c, q, lens, 4)
    c.k[c.table[b, t // 64], (t % 64) * 64:(t % 64 + 1) * 64] = 0
    for h in range(4):
        if np.all(np.isnan(out[b, h])):
            continue
        assert q[b, h, 9] * bad < 0
        p = np.array([x for x in range(n) if x != t])
        k = np.stack([O.bf16_to_f32(c.slot(c.k, c.table[b, x // 64], 0, x % 64)) for x in p]).astype(np.float64)
        v = np.stack([O.bf16_to_f32(c.slot(c.v, c.table[b, x // 64], 0, x % 64)) for x in p]).astype(np.float64)
        s = (k @ q[b, h].astype(np.float64)) * 0.125
        w = np.exp(s - s.max())
        _, bound = attn64(c, q[:, h:h + 1], lens, 1, 0.125)
        within(out[b, h], (w / w.sum()) @ v, bound[b, 0], "without it")
