"""GPU: sums of table rows that codes name, and the gradient of the tables, through the C ABI, against plain forms in 64 bits
(codes_ref.py)."""
import numpy as np
import pytest

import codes_ref as Q
import scores_ref as R

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    import vq_amd
    c = vq_amd.Context(0)
    yield c
    c.close()


def held(ctx, x, ld, offset=0, fill=np.nan):
    """Packed rows `ld` elements apart, `offset` elements into an array that holds something else around them: (array, address)."""
    n, k = x.shape
    a = np.full(offset + n * ld + 3, 0x7FFF if x.dtype == np.uint16 else fill).astype(x.dtype)
    a[offset:offset + n * ld].reshape(n, ld)[:, :k] = x
    d = ctx.to_device(a)
    return d, d.ptr + offset * x.itemsize


def device_codes(ctx, codes, nbytes, stride, offset=0):
    n, m = codes.shape
    a = np.full(offset + n * stride + 1, 1, Q.CODES[nbytes])
    a[offset:offset + n * stride].reshape(n, stride)[:, :m] = codes.astype(Q.CODES[nbytes])
    d = ctx.to_device(a)
    return d, d.ptr + offset * nbytes


def output(ctx, shape, kind, ld, offset=0, values=None):
    """An array of 7s with room for the rows, or with these values there; (array, address, what it holds)."""
    n, dim = shape
    a = R.pack(np.full(offset + n * ld + 5, 7.0), kind)
    if values is not None:
        a[offset:offset + n * ld].reshape(n, ld)[:, :dim] = values
    d = ctx.to_device(a)
    return d, d.ptr + offset * a.itemsize, a


def rows_of(d, before, shape, ld, offset, kind):
    """The rows of an output, all else in it being as before."""
    n, dim = shape
    got = d.download()
    rows = got[offset:offset + n * ld].reshape(n, ld)[:, :dim].copy()
    rest = got.copy()
    rest[offset:offset + n * ld].reshape(n, ld)[:, :dim] = before[offset:offset + n * ld].reshape(n, ld)[:, :dim]
    assert np.array_equal(rest.view(np.uint8), before.view(np.uint8))
    return rows


def near(got, want, tol):
    assert np.array_equal(np.isnan(got), np.isnan(want))
    with np.errstate(invalid="ignore"):
        ok = np.isnan(want) | (got == want) | (np.abs(got - want) <= tol)
    assert ok.all(), (np.argwhere(~ok)[:3], got[~ok][:3], want[~ok][:3], tol[~ok][:3])


SHAPES = [  # n, m, k, dim
    (1, 1, 1, 1), (1, 1, 16, 5), (3, 1, 300, 8), (7, 2, 5, 9), (16, 1, 1000, 1280), (65, 4, 33, 100), (257, 8, 256, 24), (1000, 1, 70000, 17), (33, 3, 64, 2049),
    (5, 64, 20, 40), (4099, 5, 777, 130), (2, 1, 40, 5000), (759, 2, 12388, 75), (1024, 1, 20000, 33), (900, 1, 30011, 3),
]


@pytest.mark.parametrize("kind,out", [("f32", "f32"), ("f32", "bf16"), ("f16", "f16"), ("f16", "f32"), ("bf16", "bf16"), ("bf16", "f32")])
@pytest.mark.parametrize("n,m,k,dim", SHAPES + [(20000, 5, 300, 200), (20001, 4, 700, 1030), (3000, 13, 512, 1000)])  # two pieces a lane; columns by XCD
def test_embed(ctx, n, m, k, dim, kind, out):
    rng = np.random.default_rng(n + dim)
    table = R.pack(rng.standard_normal((m * k, dim)), kind)
    nbytes = 1 if k <= 256 and n % 2 else 2 if k <= 65536 and n % 3 else 4
    codes = rng.integers(0, k, (n, m))
    if nbytes == 4:
        codes[rng.random((n, m)) < 0.2] = -1
        codes[n // 2, m - 1] = k + 3
    pad, offset, scale = n % 4, dim % 3, 1.0 if n == 1 else -2.75
    dt, pt = held(ctx, table, dim + pad, offset)
    dc, pc = device_codes(ctx, codes, nbytes, m + pad, 1)
    do, po, before = output(ctx, (n, dim), out, dim + offset, pad)
    ctx.code_embed(kind, pt, k, dim + pad, dim, m, nbytes, pc, n, m + pad, scale, out, po, dim + offset)
    got = R.unpack(rows_of(do, before, (n, dim), dim + offset, pad, out), out)
    want, err = Q.embed(R.unpack(table, kind).reshape(m, k, dim), codes, scale)
    near(got, want, Q.rounded(want, err, out))


def _grad(ctx, rng, n, m, k, dim, kind, out, codes, nbytes, accumulate=False, pad=0, offset=0, scale=1.25, again=True):
    g = R.pack(rng.standard_normal((n, dim)), kind)
    old = R.pack(rng.standard_normal((m * k, dim)), out)
    dg, pg = held(ctx, g, dim + pad, offset)
    dc, pc = device_codes(ctx, codes, nbytes, m + pad, 1)

    def call():
        do, po, before = output(ctx, (m * k, dim), out, dim + offset, pad, old)
        ctx.code_embed_grad(kind, pg, n, dim + pad, dim, m, nbytes, pc, m + pad, scale, k, accumulate, out, po, dim + offset)
        return rows_of(do, before, (m * k, dim), dim + offset, pad, out)

    rows = call()
    want, err = Q.embed_grad(R.unpack(g, kind), codes, scale, k, R.unpack(old, out).reshape(m, k, dim) if accumulate else None)
    got = R.unpack(rows, out).reshape(m, k, dim)
    near(got, want, Q.rounded(want, err, out))
    if accumulate:  # rows that no position names are as they were
        for s in range(m):
            gone = np.setdiff1d(np.arange(k), codes[:, s])
            assert np.array_equal(rows.reshape(m, k, dim)[s, gone], old.reshape(m, k, dim)[s, gone])
    if again:
        assert np.array_equal(rows, call())
    return rows


@pytest.mark.parametrize("kind,out", [("f32", "f32"), ("f32", "f16"), ("f16", "f16"), ("f16", "f32"), ("bf16", "bf16"), ("bf16", "f32")])
@pytest.mark.parametrize("accumulate", [False, True])
@pytest.mark.parametrize("n,m,k,dim", SHAPES)
def test_embed_grad(ctx, n, m, k, dim, kind, out, accumulate):
    rng = np.random.default_rng(n * 7 + dim)
    nbytes = 1 if k <= 256 and n % 2 else 2 if k <= 65536 and n % 3 else 4
    codes = rng.integers(0, k, (n, m))
    if nbytes == 4:
        codes[rng.random((n, m)) < 0.2] = -1
        codes[n // 2, m - 1] = k + 3
    _grad(ctx, rng, n, m, k, dim, kind, out, codes, nbytes, accumulate, n % 4, dim % 3, again=dim < 1000)


# numbers of members around the lines between one group of lanes, a workgroup and several workgroups per code
@pytest.mark.parametrize("kind", R.TYPES)
@pytest.mark.parametrize("members", [0, 1, 2, 7, 8, 9, 31, 32, 33, 64, 65, 511, 1023, 1024, 1025, 1500, 2048, 2049, 5000])
def test_members_of_a_code(ctx, members, kind):
    """One code with as many positions, scattered among others, at both ends of the codes' range and of the lists."""
    rng = np.random.default_rng(members)
    k, dim, n = 70, 19, members + 300
    for code in (0, 31, k - 1):
        codes = rng.integers(0, k, (n, 1))
        codes[codes == code] = (code + 1) % k
        codes[rng.permutation(n)[:members], 0] = code
        _grad(ctx, rng, n, 1, k, dim, kind, "f32", codes, 1, accumulate=code == 31)


@pytest.mark.parametrize("n", [1, 2, 63, 64, 65, 1024, 1025, 3000, 20000])
def test_all_positions_of_one_code(ctx, n):
    rng = np.random.default_rng(n)
    for k, code in ((1, 0), (300, 299), (3000, 5)):
        codes = np.full((n, 2), code)
        codes[n // 2:, 1] = 0
        _grad(ctx, rng, n, 2, k, 33, "bf16", "f32", codes, 2)


def test_several_long_codes_side_by_side(ctx):
    """Codes of more than a piece of the list each, their lists beginning and ending anywhere in the pieces."""
    rng = np.random.default_rng(9)
    counts = [1025, 1024, 3000, 1, 1100, 5, 2047, 1026, 0, 1500]
    codes = rng.permutation(np.repeat(np.arange(len(counts)), counts))[:, None]
    for out in R.TYPES:
        _grad(ctx, rng, codes.shape[0], 1, len(counts), 70, "f32", out, codes, 4, accumulate=out == "bf16")


def test_positions_without_a_code(ctx):
    rng = np.random.default_rng(1)
    codes = np.full((700, 2), -1)
    rows = _grad(ctx, rng, 700, 2, 37, 50, "f32", "f32", codes, 4)
    assert not rows.any()
    codes[:, 0] = 1 << 30  # none of the k
    codes[:, 1] = -(1 << 31)
    assert not _grad(ctx, rng, 700, 2, 37, 50, "f32", "f32", codes, 4).any()
    _grad(ctx, rng, 700, 2, 37, 50, "f32", "f32", codes, 4, accumulate=True)


def test_no_positions(ctx):
    """Without positions the gradient is zero and written as such, or left as it is; no row is read or written by the lookup."""
    g = ctx.to_device(np.full((6, 5), 3, np.float32))
    ctx.code_embed_grad("f32", None, 0, 5, 5, 2, 4, None, 2, 1.0, 3, True, "f32", g, 5)
    assert (g.download() == 3).all()
    ctx.code_embed_grad("f32", None, 0, 5, 5, 2, 4, None, 2, 1.0, 3, False, "f32", g, 5)
    assert not g.download().any()
    ctx.code_embed("f32", None, 3, 5, 5, 2, 4, None, 0, 2, 1.0, "f32", None, 5)


def test_values_that_are_no_numbers(ctx):
    """A NaN or an infinity of a row reaches the rows that have it in their sum, and no other."""
    rng = np.random.default_rng(2)
    n, k, dim = 500, 40, 21
    g = rng.standard_normal((n, dim)).astype(np.float32)
    g[3, 5], g[100, 20], g[400, 0] = np.nan, np.inf, -np.inf
    codes = rng.integers(0, k, (n, 1))
    dg, dc, do = ctx.to_device(g), ctx.to_device(codes.astype(np.uint8)), ctx.empty((k, dim), np.float32)
    ctx.code_embed_grad("f32", dg, n, dim, dim, 1, 1, dc, 1, 1.0, k, False, "f32", do, dim)
    got = do.download()
    want, _ = Q.embed_grad(g.astype(np.float64), codes, 1.0, k)
    assert np.array_equal(np.isfinite(got), np.isfinite(want[0]))
    back = ctx.empty((n, dim), np.float32)
    ctx.code_embed("f32", do, k, dim, dim, 1, 1, dc, n, 1, 1.0, "f32", back, dim)
    assert np.array_equal(back.download().view(np.uint32), got[codes[:, 0]].view(np.uint32))


def test_gradient_against_differences(ctx):
    """The change of a loss with the table, through the kernels both ways: the loss is linear, so its difference is exact but for rounding."""
    rng = np.random.default_rng(8)
    n, m, k, dim, scale = 300, 2, 50, 12, 0.5
    t, dt = rng.standard_normal((m * k, dim)).astype(np.float32), rng.standard_normal((m * k, dim)).astype(np.float32)
    w, codes = rng.standard_normal((n, dim)).astype(np.float32), rng.integers(0, k, (n, m)).astype(np.uint8)
    dc, out, grad = ctx.to_device(codes), ctx.empty((n, dim), np.float32), ctx.empty((m * k, dim), np.float32)

    def loss(table):
        d = ctx.to_device(table)
        ctx.code_embed("f32", d, k, dim, dim, m, 1, dc, n, m, scale, "f32", out, dim)
        return (out.download().astype(np.float64) * w).sum()
    ctx.code_embed_grad("f32", ctx.to_device(w), n, dim, dim, m, 1, dc, m, scale, k, False, "f32", grad, dim)
    size = np.abs(w).sum() * 10 * Q.U24 * 16
    assert abs(loss(t + dt) - loss(t) - (grad.download().astype(np.float64) * ((t + dt).astype(np.float64) - t)).sum()) < size
