"""xe_w8a8_rows_dev against its definition in 64 bits (tests/paged_util.py
rows64): the codes and the integer product are exact, so only the epilogue's
roundings are allowed for."""
import numpy as np
import pytest

from paged_util import put, rows64, within

pytestmark = pytest.mark.gpu


def make_weight(xe, ctx, rng, m, k, bias, norm, eps=1e-6):
    q8 = rng.integers(-127, 128, (m, k)).astype(np.int8)
    ws = rng.uniform(0.001, 0.02, m).astype(np.float32)
    b = rng.standard_normal(m).astype(np.float32) if bias else None
    w = ctx.register_weight_q8(q8, ws, b)
    gamma = beta = None
    if norm:
        gamma = (rng.standard_normal(k) * 0.2 + (0.0 if norm == 3 else 1.0)).astype(np.float32)
        beta = (rng.standard_normal(k) * 0.2).astype(np.float32)
        ctx.set_norm(w, xe.Norm(norm, gamma, beta, eps))
    return w, (q8, ws, b, norm, gamma, beta, eps)


def rows_case(xe, gpu, m, k, batch, norm=0, act=0, bias=True, add=False, post=False, res=False, want_sum=True, seed=0, x=None,
              alias=None):
    dev, ctx = gpu
    print("[case] rows %d x %d, %d rows, norm %d act %d" % (m, k, batch, norm, act), flush=True)
    rng = np.random.default_rng(seed + m + k + batch)
    w, defs = make_weight(xe, ctx, rng, m, k, bias, norm)
    if x is None:
        x = (rng.standard_normal((batch, k)) * np.where(rng.random(k) < 0.01, 30.0, 1.0)).astype(np.float32)
    outs = m // 2 if act == xe.XE_ACT_GEGLU else m
    a = rng.standard_normal((batch, k)).astype(np.float32) if add else None
    pw = (0.2 * rng.standard_normal(k)).astype(np.float32) if post else None
    r = rng.standard_normal((batch, outs)).astype(np.float32) if res else None
    bufs = {n: put(xe, dev, v) for n, v in (("x", x), ("add", a), ("post_w", pw), ("res", r)) if v is not None}
    bufs["y"] = bufs["res"] if alias == "y" else put(xe, dev, np.full((batch, outs), 9.0, np.float32))
    if want_sum:
        bufs["sum"] = bufs[alias] if alias in ("x", "add") else put(xe, dev, np.full((batch, k), 9.0, np.float32))
    ctx.w8a8_rows_dev(w, xe.W8a8Rows(batch, bufs["x"].ptr, bufs["y"].ptr, act=act,
                                     **{n: bufs[n].ptr for n in ("add", "post_w", "sum", "res") if n in bufs}))
    ctx.synchronize()
    y = bufs["y"].read(np.float32, batch * outs).reshape(batch, outs)
    want, t, bound = rows64(*defs, x, a, pw, act, r)
    if want_sum:
        got = bufs["sum"].read(np.float32, batch * k).reshape(batch, k)
        if post:
            within(got, t.astype(np.float64), 2 ** -23 * np.abs(t) + 1e-30, "sum")
        else:
            assert np.array_equal(got, t)
    within(y, want, bound, "rows")
    for b in {id(b): b for b in bufs.values()}.values():
        b.free()
    w.free()
    return y


@pytest.mark.parametrize("batch", [1, 2, 3, 8, 9, 15, 16, 17, 31, 33, 64, 65, 127, 128, 129, 200, 257, 512])
def test_batches(gpu, xe, batch):
    rows_case(xe, gpu, 200, 192, batch, norm=2, add=True)


@pytest.mark.parametrize("m,k", [(1, 16), (2, 16), (3, 48), (63, 112), (64, 128), (65, 144), (129, 1040), (255, 2064),
                                 (256, 4096), (1000, 768), (17, 8208), (40, 16384), (24, 32768)])
@pytest.mark.parametrize("batch", [1, 5, 40, 150])
def test_shapes(gpu, xe, m, k, batch):
    rows_case(xe, gpu, m, k, batch, norm=1, seed=5)


@pytest.mark.parametrize("m", [3, 4096, 4112])
@pytest.mark.parametrize("k", [16, 768, 784, 1280, 1296])
def test_few_rows(gpu, xe, m, k):
    """One launch and two, at the sizes where they change."""
    for batch in (1, 2, 7, 8, 9):
        rows_case(xe, gpu, m, k, batch, norm=1 + batch % 3, act=3, add=True, post=batch > 2, res=True, seed=3)


@pytest.mark.parametrize("m,k,batch", [(301, 720, 509), (702, 160, 511), (702, 4112, 397), (702, 8208, 197), (2102, 304, 509),
                                       (4102, 1040, 510), (8200, 8208, 449), (14402, 4112, 400), (97, 8208, 5),
                                       (97, 8208, 200)])
@pytest.mark.parametrize("act", [1, 4])
def test_larger_shapes(gpu, xe, m, k, batch, act):
    """Every form of the product, with tiles that end outside in both directions."""
    m += m % 2 if act == 4 else 0
    rows_case(xe, gpu, m, k, batch, norm=2, act=act, res=True, want_sum=False, seed=2)


@pytest.mark.parametrize("act", [0, 1, 2, 3, 4])
@pytest.mark.parametrize("batch", [1, 7, 30, 130])
@pytest.mark.parametrize("bias,res", [(True, True), (False, False)])
def test_epilogues(gpu, xe, act, batch, bias, res):
    rows_case(xe, gpu, 326, 256, batch, norm=3, act=act, bias=bias, res=res)


@pytest.mark.parametrize("norm", [0, 1, 2, 3])
@pytest.mark.parametrize("add,post", [(False, False), (True, False), (True, True)])
def test_prologues(gpu, xe, norm, add, post):
    for batch in (1, 20, 100):
        rows_case(xe, gpu, 96, 1152, batch, norm=norm, add=add, post=post, want_sum=True, act=2)
    rows_case(xe, gpu, 96, 1152, 4, norm=norm, add=add, post=post, want_sum=False)


@pytest.mark.parametrize("alias", ["x", "add", "y"])
def test_aliases(gpu, xe, alias):
    """The sum over x or over add, the result over the residual."""
    for batch in (1, 30, 140):
        rows_case(xe, gpu, 130, 272, batch, norm=2, add=True, res=True, alias=alias)


@pytest.mark.parametrize("batch", [1, 2, 30, 140])
@pytest.mark.parametrize("what", ["y is res is x", "res is sum", "sum is y", "y is add"])
def test_residual_stream_in_place(gpu, xe, batch, what):
    """The stream that a layer adds to, read and written by one call."""
    dev, ctx = gpu
    rng = np.random.default_rng(batch)
    n = 272
    w, defs = make_weight(xe, ctx, rng, n, n, True, 2)
    x, a = (rng.standard_normal((batch, n)).astype(np.float32) for _ in range(2))
    bx, ba, by, bs = (put(xe, dev, v) for v in (x, a, np.zeros_like(x), np.zeros_like(x)))
    if what == "y is res is x":
        ctx.w8a8_rows_dev(w, xe.W8a8Rows(batch, bx.ptr, bx.ptr, res=bx.ptr))
        want, _, bound = rows64(*defs, x, res=x)
        got = bx
    elif what == "res is sum":
        ctx.w8a8_rows_dev(w, xe.W8a8Rows(batch, bx.ptr, by.ptr, add=ba.ptr, sum=bs.ptr, res=bs.ptr))
        want, _, bound = rows64(*defs, x, a, res=x + a)
        got = by
    else:
        got = by if what == "sum is y" else ba
        ctx.w8a8_rows_dev(w, xe.W8a8Rows(batch, bx.ptr, got.ptr, add=ba.ptr, sum=by.ptr))
        want, _, bound = rows64(*defs, x, a)
    ctx.synchronize()
    within(got.read(np.float32, batch * n).reshape(batch, n), want, bound, what)
    w.free()
    for b in (bx, ba, by, bs):
        b.free()


def test_rows_do_not_depend_on_each_other(gpu, xe):
    """A row's result is the same alone and beside rows a thousand times larger,
    at every batch (kernels change with it)."""
    rng = np.random.default_rng(8)
    m, k = 320, 512
    x = rng.standard_normal((512, k)).astype(np.float32)
    x[1::2] *= 1000.0
    dev, ctx = gpu
    w, _ = make_weight(xe, ctx, rng, m, k, True, 0)
    bx, by = put(xe, dev, x), xe.Buf(dev, 512 * m * 4)
    got = {}
    for batch in (1, 2, 8, 9, 33, 64, 100, 129, 300, 512):
        ctx.w8a8_rows_dev(w, xe.W8a8Rows(batch, bx.ptr, by.ptr, act=xe.XE_ACT_GELU))
        ctx.synchronize()
        got[batch] = by.read(np.float32, batch * m).reshape(batch, m)
    for batch, y in got.items():
        assert np.array_equal(y.view(np.uint32), got[512][:batch].view(np.uint32)), batch
    for b in (bx, by):
        b.free()
    w.free()


def test_extreme_rows(gpu, xe):
    """Rows of zeros, of one value, of denormals, of the largest values; halves
    between codes round away from zero."""
    k = 256
    x = np.zeros((8, k), np.float32)
    x[1, 5] = -3.0
    x[2] = np.float32(1e-42)
    x[2, 0] = np.float32(-3e-42)
    x[3] = np.float32(3e38)
    x[3, ::3] = np.float32(-1e38)
    x[4, :] = np.linspace(-127, 127, k).astype(np.float32)
    x[4, 0] = 127.0
    x[5, 0] = 127.0
    x[5, 1:] = (np.arange(k - 1) % 127 + 0.5) * np.where(np.arange(k - 1) % 2, 1.0, -1.0)
    x[6] = 1e-30
    x[7] = -0.0
    rows_case(xe, gpu, 70, k, 8, x=x, want_sum=True)
    rows_case(xe, gpu, 70, k, 8, x=x, norm=2)


@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
def test_rows_that_are_no_numbers(gpu, xe, bad):
    """NaN in all outputs of that row, whatever the activation; the others as
    without it."""
    dev, ctx = gpu
    rng = np.random.default_rng(9)
    for batch in (3, 70):
        for act in range(5):
            m, k = 64, 160
            w, defs = make_weight(xe, ctx, rng, m, k, True, 2 if act % 2 else 0)
            x = rng.standard_normal((batch, k)).astype(np.float32)
            spoiled = x.copy()
            spoiled[1, 77] = bad
            outs = m // 2 if act == 4 else m
            bx, by = put(xe, dev, spoiled), xe.Buf(dev, batch * outs * 4)
            ctx.w8a8_rows_dev(w, xe.W8a8Rows(batch, bx.ptr, by.ptr, act=act))
            ctx.synchronize()
            y = by.read(np.float32, batch * outs).reshape(batch, outs)
            want, _, bound = rows64(*defs, x, act=act)
            assert np.all(np.isnan(y[1]))
            keep = np.arange(batch) != 1
            within(y[keep], want[keep], bound[keep], "beside NaN")
            bx.free(), by.free(), w.free()


def test_repeats_give_the_same_bits(gpu, xe):
    a = rows_case(xe, gpu, 1030, 2048, 300, norm=2, act=3)
    rows_case(xe, gpu, 64, 64, 1)
    b = rows_case(xe, gpu, 1030, 2048, 300, norm=2, act=3)
    assert np.array_equal(a.view(np.uint32), b.view(np.uint32))


def test_refusals_over_weights(gpu, xe):
    dev, ctx = gpu
    b = xe.Buf(dev, 1 << 16)
    odd = ctx.register_weight_q8(np.ones((3, 16), np.int8), np.ones(3, np.float32))
    wide = ctx.register_weight_q8(np.ones((1, 32784), np.int8), np.ones(1, np.float32))
    half = ctx.register_weight(np.ones((4, 16), np.float32), wdtype=xe.XE_BF16)
    tilted = ctx.register_weight_view(xe.XE_I8, 4, 16, b.ptr + 8, scale_ptr=b.ptr)
    for w, act in ((odd, xe.XE_ACT_GEGLU), (wide, 0), (half, 0), (tilted, 0)):
        with pytest.raises(xe.XdnaError):
            ctx.w8a8_rows_dev(w, xe.W8a8Rows(1, b.ptr, b.ptr, act=act))
    broken = ctx.register_weight_q8(np.ones((4, 16), np.int8), np.ones(4, np.float32))
    for norm, gamma in ((2, None), (1, np.ones(16, np.float32))):  # a norm that was refused
        with pytest.raises(xe.XdnaError):
            ctx.set_norm(broken, xe.Norm(norm, gamma, None, 1e-6))
        with pytest.raises(xe.XdnaError):
            ctx.w8a8_rows_dev(broken, xe.W8a8Rows(1, b.ptr, b.ptr))
    for w in (odd, wide, half, tilted, broken):
        w.free()
    b.free()


@pytest.mark.parametrize("batch", [1, 2, 20, 90, 300])
@pytest.mark.parametrize("off", [1, 2, 4])
def test_addresses(gpu, xe, batch, off):
    """Rows, results and a weight view's scales and bias at addresses off by 4, 8
    and 16 bytes from a multiple of 32; what lies around the results stays."""
    dev, ctx = gpu
    rng = np.random.default_rng(batch + off)
    m, k = 264, 1040
    q8 = rng.integers(-127, 128, (m, k)).astype(np.int8)
    ws, bias = rng.uniform(0.001, 0.02, m).astype(np.float32), rng.standard_normal(m).astype(np.float32)
    x, add = (rng.standard_normal((batch, k)).astype(np.float32) for _ in range(2))
    pw, res = (0.2 * rng.standard_normal(k)).astype(np.float32), rng.standard_normal((batch, m)).astype(np.float32)
    gamma = (1 + 0.2 * rng.standard_normal(k)).astype(np.float32)

    def shifted(a):
        return put(xe, dev, np.concatenate([np.full(off, 9.0, np.float32), a.reshape(-1), np.full(8, 9.0, np.float32)]))
    bufs = [shifted(a) for a in (ws, bias, x, add, pw, res, np.zeros((batch, k), np.float32), np.zeros((batch, m), np.float32))]
    bw = put(xe, dev, q8)
    pws, pbias, px, padd, ppost, pres, psum, py = (b.ptr + 4 * off for b in bufs)
    w = ctx.register_weight_view(xe.XE_I8, m, k, bw.ptr, scale_ptr=pws, bias_ptr=pbias)
    ctx.set_norm(w, xe.Norm(2, gamma, np.zeros(k, np.float32), 1e-6))
    ctx.w8a8_rows_dev(w, xe.W8a8Rows(batch, px, py, act=xe.XE_ACT_RELU, add=padd, post_w=ppost, sum=psum, res=pres))
    ctx.synchronize()
    want, t, bound = rows64(q8, ws, bias, 2, gamma, None, 1e-6, x, add, pw, 1, res)
    for b, n, check in ((bufs[7], batch * m, lambda g: within(g.reshape(batch, m), want, bound, "rows")),
                        (bufs[6], batch * k, lambda g: within(g.reshape(batch, k), t.astype(np.float64), 2 ** -23 * np.abs(t) + 1e-30, "sum"))):
        got = b.read(np.float32, off + n + 8)
        assert np.all(got[:off] == 9.0) and np.all(got[off + n:] == 9.0)
        check(got[off:off + n])
    w.free()
    for b in (*bufs, bw):
        b.free()
