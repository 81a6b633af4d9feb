"""GPU: rows to 8-bit integers and 8-bit scores, through the C ABI, against plain forms in 64 bits (scores_ref.py)."""
import numpy as np
import pytest

import scores_ref as R

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    import vq_amd
    c = vq_amd.Context(0)
    yield c
    c.close()


def _up(ctx, flat, offset):
    """An array that begins `offset` elements into an allocation: (array to keep, address)."""
    d = ctx.to_device(np.concatenate([np.zeros(offset, flat.dtype), flat.reshape(-1)]))
    return d, d.ptr + offset * flat.itemsize


def _quantize(ctx, x, kind, ld_pad=0, q_pad=0, offset=0, q_offset=0):
    """rows_i8 of packed values; what lies around the rows has to stay."""
    n, dim = x.shape
    held = np.full((n, dim + ld_pad), 77, x.dtype)
    held[:, :dim] = x
    dx, px = _up(ctx, held, offset)
    dq, ds = ctx.to_device(np.full(q_offset + (n + 1) * (dim + q_pad), 99, np.int8)), ctx.to_device(np.full(n + 1, -5, np.float32))
    ctx.rows_i8(kind, px, n, dim + ld_pad, dim, dq.ptr + q_offset, dim + q_pad, ds)
    q, s = dq.download(), ds.download()
    assert (q[:q_offset] == 99).all() and s[n] == -5
    q = q[q_offset:].reshape(n + 1, dim + q_pad)
    assert (q[n] == 99).all() and (q[:, dim:] == 99).all()
    return q[:n, :dim], s[:n]


@pytest.mark.parametrize("kind", R.TYPES)
@pytest.mark.parametrize("n,dim", [(1, 1), (1, 128), (3, 7), (5, 16), (64, 17), (65, 63), (130, 64), (7, 255), (33, 256), (4, 1000), (2, 1280),
                                   (3, 4099), (2, 8192), (1, 30011), (4097, 24)])
def test_rows(ctx, kind, n, dim):
    rng = np.random.default_rng([n, dim])
    x = R.pack(rng.standard_normal((n, dim)) * np.exp(rng.uniform(-20, 5, (n, 1)) if kind != "f16" else rng.uniform(-3, 5, (n, 1))), kind)
    want = R.rows_i8(R.unpack(x, kind))
    for around in (dict(), dict(ld_pad=3, q_pad=5, offset=1, q_offset=3)):
        q, s = _quantize(ctx, x, kind, **around)
        assert np.array_equal(s.view(np.uint32), want[1].view(np.uint32))
        assert np.array_equal(q, want[0])


def test_rows_on_the_borders(ctx):
    """Quotients that are ties, or a last bit off one, at every integer; scales down to the smallest."""
    rows = []
    for scale in (1.0, 3.0, 0.7, 1.1e-7, 3e37 / 127, 1.5e-38, 3e-39, 7e-45, 1.4e-45):
        s = np.float32(scale)
        top = np.float32(s * np.float32(127))
        ties = ((np.arange(-127, 127) + 0.5) * float(s)).astype(np.float32)
        row = np.concatenate([ties, np.nextafter(ties, np.float32(np.inf)), np.nextafter(ties, np.float32(-np.inf))])
        rows.append(np.concatenate([[top], np.clip(row, -top, top)]).astype(np.float32))
    x = np.stack(rows)
    q, s = _quantize(ctx, x, "f32")
    wq, ws = R.rows_i8(x.astype(np.float64))
    assert np.array_equal(s.view(np.uint32), ws.view(np.uint32))
    assert np.array_equal(q, wq)


@pytest.mark.parametrize("kind", R.TYPES)
def test_rows_without_a_scale(ctx, kind):
    x = np.zeros((6, 70), np.float32)
    x[1, 69], x[2, 3], x[3, 64] = np.inf, np.nan, -np.inf
    x[4] = np.linspace(-2, 2, 70)
    x[5] = 1e-44  # (zero in binary16 and bfloat16's nearest subnormal; the scale is zero everywhere)
    q, s = _quantize(ctx, R.pack(x, kind), kind)
    wq, ws = R.rows_i8(R.unpack(R.pack(x, kind), kind))
    assert np.isnan(s[1:4]).all() and s[0] == 0 and not q[:4].any() and np.array_equal(s, ws, equal_nan=True) and np.array_equal(q, wq)


def _scores(ctx, rng, n, dim, k, kind, bias=True, ldx=0, ldw=0, ldo=0, offset=0, worst=False):
    x, w = rng.integers(-127, 128, (n, dim + ldx)).astype(np.int8), rng.integers(-127, 128, (k, dim + ldw)).astype(np.int8)
    if worst:
        x[:], w[:] = -128, rng.choice([-128, 127], (k, 1))
    xs, ws = rng.uniform(0.001, 0.1, n).astype(np.float32), rng.uniform(0.001, 0.1, k).astype(np.float32)
    b = rng.standard_normal(k).astype(np.float32) if bias else None
    (dx, px), (dw, pw) = _up(ctx, x, offset), _up(ctx, w, offset)
    dxs, dws, db = ctx.to_device(xs), ctx.to_device(ws), ctx.to_device(b) if bias else None
    blank = R.pack(np.full((n + 1, k + ldo), -3.0), kind)
    do, po = _up(ctx, blank, offset)
    ctx.scores_i8(px, dxs, n, dim + ldx, pw, dws, k, dim + ldw, dim, db, kind, po, k + ldo)
    out = do.download()
    assert (R.unpack(out[:offset], kind) == 0).all()
    out = R.unpack(out[offset:].reshape(n + 1, k + ldo), kind)
    assert (out[n] == -3).all() and (out[:, k:] == -3).all()  # what lies around the scores stays
    want, tol = R.scores(x[:, :dim], xs, w[:, :dim], ws, b, kind)
    if kind == "f16":
        far = np.abs(want) > 65504
        assert np.isinf(out[:n, :k][np.abs(want) > 65536]).all()
        assert (np.abs(out[:n, :k] - want) <= tol)[~far].all()
    else:
        assert (np.abs(out[:n, :k] - want) <= tol).all()


SIZES = [(1, 1, 1), (1, 128, 256), (1, 16, 17), (2, 15, 3), (3, 64, 65), (7, 65, 100), (16, 1280, 333), (17, 100, 1000), (31, 127, 64), (32, 768, 1024),
         (33, 129, 129), (48, 1000, 48), (64, 256, 64), (65, 200, 513), (100, 1, 100), (127, 31, 255), (128, 128, 128), (129, 1024, 257), (255, 96, 300),
         (256, 512, 256), (257, 1000, 777), (300, 4099, 40), (513, 640, 1025), (1000, 17, 2000), (2049, 256, 5), (5000, 128, 256), (9, 8192, 700), (700, 8192, 9)]


@pytest.mark.parametrize("kind", R.TYPES)
@pytest.mark.parametrize("n,dim,k", SIZES)
def test_scores(ctx, kind, n, dim, k):
    rng = np.random.default_rng([n, dim, k])
    _scores(ctx, rng, n, dim, k, kind)                                                     # rows one after the other
    _scores(ctx, rng, n, dim, k, kind, bias=False, ldx=-dim % 16 + 16, ldw=-dim % 16, ldo=8)  # aligned, bytes that are not zero behind each row


@pytest.mark.parametrize("kind", R.TYPES)
@pytest.mark.parametrize("n,dim,k", [(1, 100, 40), (5, 77, 300), (40, 128, 130), (150, 333, 200), (300, 256, 300)])
def test_scores_any_place(ctx, kind, n, dim, k):
    rng = np.random.default_rng([n, dim, k, 1])
    _scores(ctx, rng, n, dim, k, kind, ldx=1, ldw=3, ldo=1, offset=1)
    _scores(ctx, rng, n, dim, k, kind, ldx=16, ldw=5, ldo=3, offset=5)


@pytest.mark.parametrize("ldx,ldw,offset", [(1, 0, 0), (-1037 % 16, 3, 0), (0, -1037 % 16, 0), (-1037 % 16, -1037 % 16, 4), (7, 9, 1)])
def test_scores_copied_to_aligned_rows(ctx, ldx, ldw, offset):
    """More than 2^28 to multiply: rows, codes or both at strides or addresses that are not aligned."""
    _scores(ctx, np.random.default_rng(6), 520, 1037, 530, "f32", ldx=ldx, ldw=ldw, offset=offset)


@pytest.mark.parametrize("n,dim,k", [(1, 131071, 5), (20, 131071, 20), (200, 131071, 130)])
def test_scores_longest_rows(ctx, n, dim, k):
    """The largest sums there are: 131,071 products of -128 with itself, 1023 below 2^31."""
    _scores(ctx, np.random.default_rng(3), n, dim, k, "f32", worst=True)
    _scores(ctx, np.random.default_rng(3), n, dim, k, "f32", ldx=1, ldw=1, worst=True)


def test_scores_of_rows_without_a_scale(ctx):
    n, dim, k = 20, 64, 70
    x, xs = ctx.to_device(np.zeros((n, dim), np.int8)), ctx.to_device(np.where(np.arange(n) % 3 == 0, np.nan, 0.0).astype(np.float32))
    w, ws = ctx.to_device(np.ones((k, dim), np.int8)), ctx.to_device(np.ones(k, np.float32))
    out = ctx.empty((n, k), np.float32)
    ctx.scores_i8(x, xs, n, dim, w, ws, k, dim, dim, None, "f32", out, k)
    got = out.download()
    assert np.isnan(got[::3]).all() and (np.delete(got, np.s_[::3], axis=0) == 0).all()


def test_many_rows(ctx):
    """More rows than one grid dimension holds tiles of."""
    rng = np.random.default_rng(9)
    n, dim, k = 65535 * 64 + 777, 3, 2
    x, w = rng.integers(-127, 128, (n, dim)).astype(np.int8), rng.integers(-127, 128, (k, dim)).astype(np.int8)
    xs, ws = rng.uniform(0.5, 1, n).astype(np.float32), np.ones(k, np.float32)
    out = ctx.empty((n, k), np.float32)
    ctx.scores_i8(ctx.to_device(x), ctx.to_device(xs), n, dim, ctx.to_device(w), ctx.to_device(ws), k, dim, dim, None, "f32", out, k)
    want, tol = R.scores(x, xs, w, ws, None, "f32")
    assert (np.abs(out.download() - want) <= tol).all()


def test_refusals_leave_the_context_usable(ctx):
    import vq_amd
    x = ctx.to_device(np.ones((4, 16), np.int8))
    s, out = ctx.to_device(np.ones(4, np.float32)), ctx.empty((4, 4), np.float32)
    with pytest.raises(vq_amd.VqError) as e:
        ctx.scores_i8(x, s, 4, 15, x, s, 4, 16, 16, None, "f32", out, 4)
    assert e.value.code == vq_amd._ffi.ERR_INVALID_ARG and "stride" in str(e.value)
    with pytest.raises(vq_amd.VqError) as e:
        ctx.rows_i8(vq_amd.F32, out, 4, 4, 131072, x, 16, s)
    assert e.value.code == vq_amd._ffi.ERR_UNSUPPORTED
    ctx.scores_i8(x, s, 4, 16, x, s, 4, 16, 16, None, vq_amd.F32, out, 4)
    assert (out.download() == 16).all()


def test_order_of_the_distances(ctx):
    """With the bias -|c|^2 / 2 the largest score is the nearest codeword's, as vq_assign finds it, wherever the two best
    distances are further apart than the 8-bit rounding of rows and codewords reaches."""
    import vq_amd
    rng = np.random.default_rng(4)
    n, dim, k = 500, 64, 256
    cb = rng.standard_normal((k, dim)).astype(np.float32)
    x = (cb[rng.integers(0, k, n)] + 0.05 * rng.standard_normal((n, dim))).astype(np.float32)
    dx, dcb, codes = ctx.to_device(x), ctx.to_device(cb), ctx.empty((n, 1), np.uint8)
    ctx.assign(vq_amd.SQEUCLIDEAN, dx, n, dim, 1, dim, k, dcb, codes)
    xq, wq = ctx.empty((n, dim), np.int8), ctx.empty((k, dim), np.int8)
    xs, ws, out = ctx.empty(n, np.float32), ctx.empty(k, np.float32), ctx.empty((n, k), np.float32)
    ctx.rows_i8("f32", dx, n, dim, dim, xq, dim, xs)
    ctx.rows_i8("f32", dcb, k, dim, dim, wq, dim, ws)
    bias = ctx.to_device((-0.5 * (cb.astype(np.float64) ** 2).sum(1)).astype(np.float32))
    ctx.scores_i8(xq, xs, n, dim, wq, ws, k, dim, dim, bias, "f32", out, k)
    # a component is off by half a scale at most, so a score by |dx| |c|_1 + |x|_1 |dw| + dim |dx| |dw|
    hx, hw = xs.download().astype(np.float64) / 2, ws.download().astype(np.float64) / 2
    off = (hx[:, None] * np.abs(cb).sum(1) + np.abs(x).sum(1)[:, None] * hw + dim * hx[:, None] * hw).max(1) + 1e-3
    exact = x.astype(np.float64) @ cb.astype(np.float64).T - 0.5 * (cb.astype(np.float64) ** 2).sum(1)
    two = np.sort(exact, axis=1)[:, -2:]
    clear = two[:, 1] - two[:, 0] > 2 * off
    assert clear.sum() > 100
    assert np.array_equal(out.download().argmax(1)[clear], codes.download()[clear, 0])
