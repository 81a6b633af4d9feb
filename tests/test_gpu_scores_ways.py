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
