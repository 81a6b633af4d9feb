"""GPU: 8-bit scores by every way that aligned rows go, against the exact sums (scores_ref.py)."""
import numpy as np
import pytest

import scores_ref as R
from scores_sizes import SIZES

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    import vq_amd
    c = vq_amd.Context(0)
    yield c
    c.close()


@pytest.mark.parametrize("n,dim,k", [s for way in SIZES.values() for s in way])
def test_ways(ctx, n, dim, k):
    """Rows padded to 16 bytes, with bytes that are not zero behind their components; scores whose rows are whole lines of 128
    bytes, which pass the caches, and not; with a bias and without.  The 16-bit scores are the f32 ones, rounded once."""
    rng = np.random.default_rng([n, dim, k])
    ld, whole = (dim + 15) // 16 * 16, -(-k // 64) * 64 + 64
    x, w = rng.integers(-128, 128, (n, ld + 16)).astype(np.int8), rng.integers(-128, 128, (k, ld)).astype(np.int8)
    xs, ws = rng.uniform(0.001, 0.01, n).astype(np.float32), rng.uniform(0.001, 0.01, k).astype(np.float32)
    bias = rng.standard_normal(k).astype(np.float32)
    dx, dw, dxs, dws, db = (ctx.to_device(a) for a in (x, w, xs, ws, bias))
    y0 = (x[:, :dim].astype(np.float64) @ w[:, :dim].astype(np.float64).T) * xs.astype(np.float64)[:, None] * ws.astype(np.float64)

    def call(b, kind, ld_out):
        out = ctx.to_device(np.full((n + 1, ld_out), 7, np.uint32 if kind == "f32" else np.uint16))
        assert out.ptr % 128 == 0
        ctx.scores_i8(dx, dxs, n, ld + 16, dw, dws, k, ld, dim, b, kind, out, ld_out)
        raw = out.download()
        out.free()
        assert (raw[n] == 7).all() and (raw[:, k:] == 7).all()
        return raw[:n, :k]
    for b, lds in ((db, (k, whole, k, whole)), (None, (whole, k, whole, k))):
        f32 = call(b, "f32", lds[0])
        assert np.array_equal(f32, call(b, "f32", lds[1]))
        f32 = np.ascontiguousarray(f32).view(np.float32)
        y = y0 + bias if b is not None else y0
        # the conversion of the sum, two products and the sum with the bias are rounded once each
        assert (np.abs(f32 - y) <= 1.01 * (3.01 * R.U24 * np.abs(y0) + R.U24 * np.abs(y))).all()
        assert np.array_equal(call(b, "f16", lds[2]), R.pack(f32, "f16").view(np.uint16))
        assert np.array_equal(call(b, "bf16", lds[3]), R.pack(f32, "bf16"))


@pytest.mark.parametrize("n,dim,k", [way[0] for way in SIZES.values()])
def test_rows_that_are_not_aligned_score_the_same(ctx, n, dim, k):
    """The copy to aligned rows, the kernel for any place and the ways of aligned rows: the same bits."""
    rng = np.random.default_rng([n, dim, k, 2])
    ld = (dim + 15) // 16 * 16
    x, w = rng.integers(-128, 128, (n, dim)).astype(np.int8), rng.integers(-128, 128, (k, dim)).astype(np.int8)
    wide = np.full((n, ld), 9, np.int8)
    wide[:, :dim] = x
    codes = np.full((k, ld), 11, np.int8)
    codes[:, :dim] = w
    xs, ws = ctx.to_device(rng.uniform(0.001, 0.01, n).astype(np.float32)), ctx.to_device(rng.uniform(-0.01, 0.01, k).astype(np.float32))
    a, b = ctx.empty((n, k), np.float32), ctx.empty((n, k), np.float32)
    ctx.scores_i8(ctx.to_device(wide), xs, n, ld, ctx.to_device(codes), ws, k, ld, dim, None, "f32", a, k)
    away = ctx.to_device(np.concatenate([np.zeros(1, np.int8), x.reshape(-1)]))
    ctx.scores_i8(away.ptr + 1, xs, n, dim, ctx.to_device(w), ws, k, dim, dim, None, "f32", b, k)
    assert np.array_equal(a.download().view(np.uint32), b.download().view(np.uint32))


@pytest.mark.parametrize("n,dim,k", [way[0] for way in SIZES.values()])
@pytest.mark.parametrize("kind", R.TYPES)
def test_sign_of_a_zero_score(ctx, kind, n, dim, k):
    """Without a bias nothing is added: a sum of zero under a negative scale is -0, by every way; with a bias of 0 it is 0."""
    ld = (dim + 15) // 16 * 16
    x, w = ctx.to_device(np.zeros((n, ld), np.int8)), ctx.to_device(np.zeros((k, ld), np.int8))
    sign = np.where(np.arange(k) % 3 == 0, -1.0, 1.0).astype(np.float32)
    xs, ws, none = ctx.to_device(np.ones(n, np.float32)), ctx.to_device(sign), ctx.to_device(np.zeros(k, np.float32))
    out = ctx.to_device(R.pack(np.full((n, k), -3.0, np.float32), kind))
    bit = np.uint32(1 << 31) if kind == "f32" else np.uint16(1 << 15)
    for ptr in (x.ptr, x.ptr + 1):  # (the second: rows that are not aligned, the last one 15 bytes shorter than there are)
        rows = n if ptr == x.ptr else n - 1
        ctx.scores_i8(ptr, xs, rows, ld, w, ws, k, ld, dim, None, kind, out, k)
        got = out.download()[:rows].view(bit.dtype)
        assert (got == np.where(sign < 0, bit, bit.dtype.type(0))).all()
        ctx.scores_i8(ptr, xs, rows, ld, w, ws, k, ld, dim, none, kind, out, k)
        assert not out.download()[:rows].view(bit.dtype).any()
