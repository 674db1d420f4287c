"""A weight whose norm was refused: every call that would apply it is refused on
the host, whichever kernel its rows take, until a norm is set."""
import numpy as np
import pytest

from paged_util import put

pytestmark = pytest.mark.gpu

# from one row (the GEMV) to the most (the GEMM, over row planes and not)
BATCHES = [1, 8, 9, 64, 65, 200, 512]


def weights(xe, ctx, rng, m, k):
    w = (0.05 * rng.standard_normal((m, k))).astype(np.float32)
    return [ctx.register_weight(w, wdtype=t) for t in (xe.XE_BF16, xe.XE_I8, xe.XE_BFP16)]


@pytest.mark.parametrize("kind", [1, 2, 3])
def test_refused_norm(gpu, xe, kind):
    dev, ctx = gpu
    rng = np.random.default_rng(kind)
    m, k = 256, 512
    gamma, beta = rng.standard_normal(k).astype(np.float32), rng.standard_normal(k).astype(np.float32)
    x = rng.standard_normal((max(BATCHES), k)).astype(np.float32)
    bx, by = put(xe, dev, x), xe.Buf(dev, max(BATCHES) * m * 4)
    for w in weights(xe, ctx, rng, m, k):
        for had_one in (False, True):
            if had_one:
                ctx.set_norm(w, xe.Norm(kind, gamma, beta, 1e-5))
            with pytest.raises(xe.XdnaError):
                ctx.set_norm(w, xe.Norm(kind, gamma if kind == xe.XE_NORM_LN else None, None, 1e-5))
            for batch in BATCHES:
                with pytest.raises(xe.XdnaError, match="lacks gamma or beta"):
                    ctx.gemv_dev(w, bx, batch, by)
                with pytest.raises(xe.XdnaError, match="lacks gamma or beta"):
                    ctx.fused_norm_gemv(w, x[:batch])
            if w.wdtype == xe.XE_I8:
                with pytest.raises(xe.XdnaError, match="lacks gamma or beta"):
                    ctx.w8a8_rows_dev(w, xe.W8a8Rows(4, bx.ptr, by.ptr))
            with pytest.raises(xe.XdnaError, match="lacks gamma or beta"):
                ctx.probe_gemv([w], bx.ptr, xe.XE_F32, 64, by.ptr, 1, eager=True)
        # a norm again, and none: as a weight that was never refused
        ctx.set_norm(w, xe.Norm(kind, gamma, beta, 1e-5))
        for batch in BATCHES:
            a = ctx.fused_norm_gemv(w, x[:batch])
            assert np.all(np.isfinite(a)) and np.any(a != 0)
        ctx.set_norm(w, xe.Norm(xe.XE_NORM_NONE, None, None, 1e-5))
        assert np.all(np.isfinite(ctx.gemv(w, x[:9])))
        w.free()
    bx.free(), by.free()


def test_unknown_norm_changes_nothing(gpu, xe):
    dev, ctx = gpu
    rng = np.random.default_rng(5)
    x, gamma = rng.standard_normal((20, 64)).astype(np.float32), rng.standard_normal(64).astype(np.float32)
    w = weights(xe, ctx, rng, 48, 64)[0]
    ctx.set_norm(w, xe.Norm.Rms(gamma))
    before = ctx.fused_norm_gemv(w, x)
    with pytest.raises(xe.XdnaError):
        ctx.set_norm(w, xe.Norm(4, gamma, None, 1e-5))
    assert np.array_equal(before, ctx.fused_norm_gemv(w, x))
    w.free()
