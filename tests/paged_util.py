"""Plain 64-bit forms of the paged cache's operators and of the int8 linears
with a scale a row, in numpy, and device buffers for their tests."""
import math

import numpy as np

import oracle_lib as O

EPS32 = 2.0 ** -24  # half a step of fp32
EPS16 = 2.0 ** -8   # half a step of bf16


class At:
    """A device address as a buffer."""

    def __init__(self, ptr):
        self.ptr = ptr


def put(xe, dev, a):
    return xe.Buf.from_array(dev, np.ascontiguousarray(a))


def f64(bits):
    return O.bf16_to_f32(bits).astype(np.float64)


class Cache:
    """A paged cache on the host and on the device: random rows in every slot,
    the pages of the streams scattered over the pool."""

    def __init__(self, xe, dev, rng, batch, max_pages, page, hkv, hd, spare=3, gap=0):
        self.xe, self.dims = xe, (batch, max_pages, page, hkv, hd)
        n = batch * max_pages + spare
        self.n_pages, self.dense = n, hkv * page * hd
        self.stride = self.dense + gap
        self.table = rng.permutation(n)[:batch * max_pages].astype(np.int32).reshape(batch, max_pages)
        self.k = O.bf16_bits(rng.standard_normal((n, self.stride)).astype(np.float32))
        self.v = O.bf16_bits(rng.standard_normal((n, self.stride)).astype(np.float32))
        self.dev = dev
        self.bufs = None

    def upload(self):
        self.bufs = [put(self.xe, self.dev, a) for a in (self.k, self.v, self.table)]
        batch, max_pages, page, hkv, hd = self.dims
        return self.xe.PagedKV(*self.bufs, self.n_pages, hkv, page, hd, batch, max_pages,
                               page_stride=0 if self.stride == self.dense else self.stride)

    def read(self):
        """(k, v) bits as the device has them."""
        return tuple(b.read(np.uint16, self.k.size).reshape(self.k.shape) for b in self.bufs[:2])

    def slot(self, bits, page, head, at):
        _, _, ps, _, hd = self.dims
        o = (head * ps + at) * hd
        return bits[page, o:o + hd]

    def free(self):
        for b in self.bufs:
            b.free()


def heads64(x, w, eps, cos, sin, pos):
    """[h, hd] heads of one row in 64 bits: RMSNorm (1 + w), rotation."""
    x = x.astype(np.float64)
    if w is not None:
        x = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * (1.0 + w.astype(np.float64))
    if cos is not None:
        half = x.shape[-1] // 2
        a, b, c, s = x[:, :half], x[:, half:], cos[pos].astype(np.float64), sin[pos].astype(np.float64)
        x = np.concatenate([a * c - b * s, b * c + a * s], -1)
    return x


def attn64(cache, q, lens, hq, scale, window=0):
    """(out [batch, hq, hd] in 64 bits, a bound of the kernel's error a value).

    The bound: scores are dot products of hd fp32 terms (hd + 4 roundings of at
    most the sum of their magnitudes) scaled and taken to base 2 (4 roundings
    of their size), each weight errs by twice that, relative, and the weighted
    sum of n values adds n + 8 roundings of at most their largest."""
    batch, max_pages, page, hkv, hd = cache.dims
    out, bound = np.zeros((batch, hq, hd)), np.zeros((batch, hq, 1))
    for b in range(batch):
        n = int(lens[b])
        lo = max(0, n - window) if window else 0
        ok = [t for t in range(lo, min(max(n, 0), max_pages * page))
              if 0 <= cache.table[b, t // page] < cache.n_pages]
        if not ok:
            continue
        for g in range(hkv):
            k = np.stack([f64(cache.slot(cache.k, cache.table[b, t // page], g, t % page)) for t in ok])
            v = np.stack([f64(cache.slot(cache.v, cache.table[b, t // page], g, t % page)) for t in ok])
            for h in range(g * (hq // hkv), (g + 1) * (hq // hkv)):
                x = q[b, h].astype(np.float64)
                s = (k @ x) * scale
                p = np.exp(s - s.max())
                out[b, h] = (p / p.sum()) @ v
                d = (hd + 4) * (np.abs(k) @ np.abs(x)).max() * abs(scale) + 4 * np.abs(s).max() + 8
                bound[b, h] = EPS32 * (2 * d + len(ok) + 8) * np.abs(v).max()
    return out, bound


def rows64(q8, ws, bias, norm, gamma, beta, eps, x, add=None, post=None, act=0, res=None):
    """(y, x + add, a bound of the kernel's error a value): codes and scales as
    defined, everything else in 64 bits.  norm: 0 none, 1 LN, 2 RMS, 3 RMS
    (1 + w); act: enum xe_act.

    The bound: the codes' product is whole; its conversion, two scales and the
    bias are four roundings of at most |acc s ws| + |bias|; an activation passes
    them on with a slope of at most 1.13 and adds 8 roundings of its size."""
    x = np.asarray(x, np.float32)
    t = x
    if add is not None:
        a = np.asarray(add, np.float32)
        if post is not None:
            a64 = a.astype(np.float64)
            inv = 1.0 / np.sqrt((a64 * a64).mean(1, keepdims=True) + float(np.float32(eps)))
            a = (a64 * inv * (1.0 + post.astype(np.float64))).astype(np.float32)
        t = x + a
    h = t.astype(np.float64)
    if norm == 1:
        h = h - h.mean(1, keepdims=True)
    if norm:
        h = h / np.sqrt((h * h).mean(1, keepdims=True) + float(np.float32(eps)))
        h = h * ((1.0 if norm == 3 else 0.0) + gamma.astype(np.float64))
    if norm == 1:
        h = h + beta.astype(np.float64)
    amax = np.abs(h).max(1)
    s = np.where(amax > 0, amax / 127.0, 1.0).astype(np.float32)
    s = np.where(s > 0, s, np.float32(1))
    r = h / s.astype(np.float64)[:, None]
    codes = np.clip(np.sign(r) * np.floor(np.abs(r) + 0.5), -127, 127)
    z = (codes @ q8.T.astype(np.float64)) * s.astype(np.float64)[:, None]
    z = np.where(np.abs(z) > float(np.finfo(np.float32).max), np.copysign(np.inf, z), z)  # held in fp32, as is the product
    z = z * ws.astype(np.float64)
    z = np.where(np.abs(z) > float(np.finfo(np.float32).max), np.copysign(np.inf, z), z)
    mag = np.abs(z)
    if bias is not None:
        z = z + bias
        mag = mag + np.abs(bias)
    err = 4 * EPS32 * mag
    erf = np.vectorize(math.erf)
    if act == 1:
        y = np.maximum(z, 0.0)
    elif act == 2:
        y = 0.5 * z * (1.0 + erf(z / math.sqrt(2.0)))
    elif act == 3:
        y = z / (1.0 + np.exp(-z))
    elif act == 4:
        g, u, eg, eu = z[:, 0::2], z[:, 1::2], err[:, 0::2], err[:, 1::2]
        f = 0.5 * g * (1.0 + np.tanh(math.sqrt(2.0 / math.pi) * (g + 0.044715 * g ** 3)))
        y = f * u
        err = (1.13 * eg + 8 * EPS32 * np.abs(g)) * np.abs(u) + eu * np.abs(f) + 2 * EPS32 * np.abs(y)
    else:
        y = z
    if act in (1, 2, 3):
        err = 1.13 * err + 8 * EPS32 * np.abs(z)
    if res is not None:
        y = y + res
        err = err + EPS32 * np.abs(y)
    return y, t, err + 1e-37


def within(got, want, bound, what=""):
    got, want, bound = np.broadcast_arrays(np.asarray(got, np.float64), want, bound)
    fine = np.isfinite(want)
    assert np.array_equal(got[~fine], want[~fine]), what
    got, want, bound = got[fine], want[fine], bound[fine]
    d = np.abs(got - want)
    assert np.all(np.isfinite(d)), what
    over = d - bound
    i = np.unravel_index(np.argmax(over), over.shape)
    assert over[i] <= 0, "%s: off by %.3g where %.3g is allowed, at %s" % (what, d[i], np.broadcast_to(bound, d.shape)[i], i)
