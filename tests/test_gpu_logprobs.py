"""GPU: log probabilities of codes, entropy, alternatives and the gradient, through the C ABI, against plain forms in 64
bits (scores_ref.py)."""
import ctypes as C

import numpy as np
import pytest

import scores_ref as R

pytestmark = pytest.mark.gpu
CODES = {1: np.uint8, 2: np.uint16, 4: np.int32}


@pytest.fixture(scope="module")
def ctx():
    import vq_amd
    c = vq_amd.Context(0)
    yield c
    c.close()


def _held(x, ld, offset):
    """Rows `ld` elements apart, `offset` elements into the array; NaN-like bytes around them."""
    n, k = x.shape
    a = np.full(offset + n * ld, 0x7FFF if x.dtype == np.uint16 else np.nan).astype(x.dtype)
    a[offset:].reshape(n, ld)[:, :k] = x
    return a


class Call:
    def __init__(self, ctx, x, kind, beta, codes, code_bytes=4, code_stride=1, top=0, pad=0, offset=0):
        """x: packed rows.  Runs the forward call and keeps everything."""
        self.ctx, self.kind, self.beta, self.n, self.k = ctx, kind, beta, *x.shape
        n, self.ld, self.offset, self.top = self.n, self.k + pad, offset, top
        self.x = R.unpack(x, kind)
        self.dev = ctx.to_device(_held(x, self.ld, offset))
        self.ptr = self.dev.ptr + offset * x.itemsize
        self.code_bytes, self.code_stride, self.codes = code_bytes, code_stride, codes
        wide = np.full(n * code_stride, 3, CODES[code_bytes])
        wide[::code_stride] = codes.astype(CODES[code_bytes])
        self.dcodes = ctx.to_device(wide)
        self.out = [ctx.to_device(np.full(n + 1, 7, np.float32)) for _ in range(4)]
        self.top_lp, self.top_code = ctx.to_device(np.full((n + 1, max(top, 1)), 7, np.float32)), ctx.to_device(np.full((n + 1, max(top, 1)), 7, np.int32))
        self.run()

    def run(self):
        self.ctx.code_logprobs(self.kind, self.ptr, self.n, self.ld, self.k, self.beta, self.code_bytes, self.dcodes, self.code_stride, self.top,
                               *self.out, self.top_lp, self.top_code)

    def check(self):
        lp, m, L, H = (o.download() for o in self.out)
        n, k = self.n, self.k
        for o in (lp, m, L, H):
            assert o[n] == 7  # behind the last row
        lp, m, L, H = lp[:n], m[:n], L[:n], H[:n]
        st = R.statistics(self.x, self.beta)
        tL, tH = R.bounds(st, k)
        none, bad, fine = st["none"], st["bad"], ~st["none"] & ~st["bad"]
        assert np.array_equal(m[~np.isnan(st["m"])], st["m"][~np.isnan(st["m"])].astype(np.float32)) and np.isnan(m[np.isnan(st["m"])]).all()
        assert (np.abs(L - st["L"])[fine] <= tL[fine]).all(), np.max(np.abs(L - st["L"])[fine] / tL[fine])
        assert (np.abs(H - st["H"])[fine] <= tH[fine]).all(), np.max(np.abs(H - st["H"])[fine] / tH[fine])
        assert np.isnan(L[bad]).all() and np.isnan(H[bad]).all() and (L[none] == -np.inf).all() and (H[none] == 0).all()
        c = self.codes.astype(np.int64)
        at = np.clip(c, 0, k - 1)
        want = st["lp"][np.arange(n), at]
        with np.errstate(invalid="ignore"):
            tol = (2 * np.abs(st["d"][np.arange(n), at]) + np.abs(want)) * R.U24 * 1.01 + tL
            near = (lp == R.f32(want)) | (np.abs(lp - want) <= tol) | (np.isnan(lp) & np.isnan(want))
        assert near[(c >= 0) & (c < k)].all()
        assert (lp[c < 0] == 0).all() and np.isnan(lp[c >= k]).all()
        if self.top:
            tl, tc = self.top_lp.download(), self.top_code.download()
            assert (tl[n] == 7).all() and (tc[n] == 7).all()
            want = R.best(self.x, self.top)
            want[bad] = -1
            assert np.array_equal(tc[:n], want)
            i, t = np.nonzero(want >= 0)
            j = want[i, t]
            tol = (2 * np.abs(st["d"][i, j]) + np.abs(st["lp"][i, j])) * R.U24 * 1.01 + tL[i]
            with np.errstate(invalid="ignore"):
                assert ((tl[i, t] == R.f32(st["lp"][i, j])) | (np.abs(tl[i, t] - st["lp"][i, j]) <= tol)).all()
            assert np.isnan(tl[:n][bad]).all() and (tl[:n][(want < 0) & ~bad[:, None]] == -np.inf).all()
        return self

    def grad(self, gl, gh, inplace=False, pad=None):
        """The backward call, checked; gl, gh: arrays or None."""
        ctx, n, k = self.ctx, self.n, self.k
        ld = self.ld if inplace or pad is None else k + pad
        dgl, dgh = (None if g is None else ctx.to_device(g.astype(np.float32)) for g in (gl, gh))
        item = 4 if self.kind == "f32" else 2
        if inplace:
            d, p, before = self.dev, self.ptr, self.dev.download()
        else:
            d = ctx.to_device(R.pack(np.full(n * ld + 1, 5.0), self.kind))
            p, before = d.ptr, d.download()
        ctx.code_logprobs_grad(self.kind, self.ptr, n, self.ld, k, self.beta, self.code_bytes, self.dcodes, self.code_stride, self.out[1], self.out[2],
                               self.out[3] if gh is not None else None, dgl, dgh, p, ld)
        raw = d.download()
        o = self.offset if inplace else 0
        got = raw[o:o + n * ld].reshape(n, ld)
        keep = before[o:o + n * ld].reshape(n, ld)
        assert np.array_equal(got[:, k:].view(np.uint8), keep[:, k:].view(np.uint8)) and np.array_equal(raw[n * ld + o:].view(np.uint8), before[n * ld + o:].view(np.uint8))
        got = R.unpack(got[:, :k], self.kind)
        m, L, H = (v.download()[:n] for v in self.out[1:])
        codes = self.codes.astype(np.int64) if gl is not None else np.full(n, -1)
        want, err = R.grad(self.x, self.beta, codes, m, L, H, gl if gl is None else gl.astype(np.float32), gh if gh is None else gh.astype(np.float32))
        tol = err + 1.01 * R.HALF_STEP[self.kind] * (np.abs(want) + err) + R.LEAST[self.kind]
        assert np.array_equal(np.isnan(got), np.isnan(want))
        ok = np.isnan(want) | (np.abs(got - want) <= tol)
        assert ok.all(), (np.argwhere(~ok)[:3], got[~ok][:3], want[~ok][:3], tol[~ok][:3])
        assert item
        return got


def _rows(rng, n, k, spread=2.5):
    return rng.standard_normal((n, k)) * spread


SIZES = [(1, 1), (1, 2), (3, 3), (2, 15), (5, 16), (4, 17), (9, 63), (7, 64), (3, 65), (33, 100), (2, 127), (6, 255), (300, 256), (5, 257), (4, 511), (3, 512),
         (2, 513), (3, 1000), (2, 1023), (5, 1024), (3, 1025), (2, 2047), (2, 2049), (3, 4095), (2, 4096), (2, 4099), (1, 8191), (2, 10007), (1, 16383), (2, 16384),
         (1, 16385), (3, 32768), (2, 50021), (1, 65535), (2, 65536), (1, 65537), (1, 131073), (1, 262144), (1, 1000003), (1000, 7), (70, 999)]


@pytest.mark.parametrize("kind", R.TYPES)
@pytest.mark.parametrize("n,k", SIZES)
def test_sizes(ctx, kind, n, k):
    rng = np.random.default_rng([n, k])
    x = R.pack(_rows(rng, n, k), kind)
    codes = rng.integers(0, k, n)
    width = 1 if k <= 256 else 2 if k <= 65536 else 4
    c = Call(ctx, x, kind, 1.0, codes, width, 1 + n % 3, top=5, pad=n % 2).check()
    c.grad(rng.standard_normal(n), rng.standard_normal(n), pad=k % 3)


@pytest.mark.parametrize("kind", R.TYPES)
@pytest.mark.parametrize("top", [0, 1, 2, 3, 8, 19, 20, 31, 32])
@pytest.mark.parametrize("n,k", [(40, 5), (33, 40), (21, 256), (3, 1500), (5, 5000), (2, 40000)])
def test_tops(ctx, kind, top, n, k):
    rng = np.random.default_rng([n, k, top])
    Call(ctx, R.pack(_rows(rng, n, k), kind), kind, 0.7, rng.integers(0, k, n), top=top).check()


@pytest.mark.parametrize("kind", R.TYPES)
@pytest.mark.parametrize("k", [5, 33, 256, 300, 700, 1024, 3000, 20000, 70001])
def test_orders_and_ties(ctx, kind, k):
    """Rows in which the alternatives are hard to come by: rising, falling, all the same, few different values, the best ones
    side by side in one thread's share, all but a few impossible, the last code the best."""
    rng = np.random.default_rng(k)
    ramp = np.linspace(-8, 8, k)
    x = np.stack([ramp, ramp[::-1], np.zeros(k), np.full(k, -3.4e38 if kind != "f16" else -65504.0), rng.integers(0, 3, k).astype(float), rng.integers(0, 2, k) * 1.0,
                  np.where(np.arange(k) // 64 == (k // 64) // 2, 5.0, 0.0) + rng.standard_normal(k) * 0.01, np.where(rng.random(k) < 3.0 / k, 1.0, -np.inf),
                  np.where(np.arange(k) == k - 1, 9.0, 1.0), np.where(np.arange(k) == 0, 9.0, -np.inf), np.where(np.arange(k) % 2 == 0, 0.0, -0.0),
                  np.where(np.arange(k) % 256 == 17, 4.0, rng.standard_normal(k)), np.full(k, -np.inf), np.where(np.arange(k) % 64 < 4, 3.0, 1.0)])
    for top in (1, 4, 32):
        Call(ctx, R.pack(x, kind), kind, 1.0, rng.integers(0, k, len(x)), top=top).check()


@pytest.mark.parametrize("kind", R.TYPES)
@pytest.mark.parametrize("n,k,top", [(30, 256, 32), (30, 200, 9), (30, 300, 32), (30, 513, 17), (30, 1100, 32), (30, 4096, 9), (30, 16500, 32), (30, 33000, 12),
                                     (16500, 132, 16), (16500, 256, 20), (16400, 256, 32), (16400, 129, 31)])
def test_floor_of_many_alternatives(ctx, kind, n, k, top):
    """More than eight alternatives per wave: scores alike in their leading bits, below zero, around zero and subnormal, fewer of
    them above -inf than asked for, in few threads, with NaN or +inf; and many short rows."""
    rng = np.random.default_rng([n, k, top])
    x = _rows(rng, n, k).astype(np.float32)
    near = rng.integers(0, 400, k)
    x[0] = np.float32(1.0) + near.astype(np.float32) * np.float32(2.0 ** -23)
    x[1] = -(np.float32(1.0) + near.astype(np.float32) * np.float32(2.0 ** -23))
    x[2] = -np.abs(x[2]) - 100
    x[3] = (near - 200) * 2.0 ** -149
    x[4] = np.where(near % 2 == 0, 0.0, -0.0)
    x[5] = np.where(np.arange(k) < top - 1, x[5], -np.inf)
    x[6] = np.where(np.arange(k) >= k - top, x[6], -np.inf)
    x[7] = np.where(np.arange(k) % 8 == 0, -3.0, -np.inf)
    x[8], x[8, ::8] = -5.0, np.nan
    x[9, k - 1] = np.inf
    x[10] = np.where(np.arange(k) // 8 < 9, 50.0 + x[10], -50.0)
    x[11] = 2.0 ** rng.integers(-30, 15, k)
    x[12] = -x[11]
    x[13] = -65504.0
    x[14] = -np.inf
    x[15] = np.where(np.arange(k) == k // 2, x[15], -np.inf)
    x[16] = np.nan
    Call(ctx, R.pack(x, kind), kind, 1.0, rng.integers(-1, k + 1, n), top=top, pad=n % 4).check()


@pytest.mark.parametrize("kind", R.TYPES)
@pytest.mark.parametrize("k", [1025, 1600, 2048, 2049, 3001, 4096])
def test_many_rows_of_a_wave(ctx, kind, k):
    """Enough rows for a wave each: ties, masks, rows with nothing left and rows of equal scores among them."""
    n = 4099
    rng = np.random.default_rng(k)
    x = rng.integers(-8, 9, (n, k)) * 0.5 if k % 2 else _rows(rng, n, k)
    x = x.astype(np.float32)
    x[::7] = np.where(rng.random((len(x[::7]), k)) < 0.5, -np.inf, x[::7])
    x[3::11] = 1.25
    x[5] = -np.inf
    x[6, :k - 3] = -np.inf
    x[8, k // 2] = np.nan
    codes = rng.integers(-1, k + 1, n)
    Call(ctx, R.pack(x, kind), kind, 0.9, codes, top=7 if k % 3 else 32).check()


@pytest.mark.parametrize("kind", R.TYPES)
@pytest.mark.parametrize("k", [1, 2, 70, 256, 1500, 9000, 40000])
def test_masks_and_codes(ctx, kind, k):
    rng = np.random.default_rng(k)
    low = -3.3e38 if kind != "f16" else -65504.0
    x = _rows(rng, 14, k)
    x[1] = -np.inf                       # nothing is left
    x[2, rng.random(k) < 0.9] = -np.inf
    x[3] = np.where(rng.random(k) < 0.5, low, x[3])  # masks of the type's lowest value
    x[4] = low
    x[5, k // 2] = np.inf
    x[6, k - 1] = np.nan
    x[7] = -np.inf
    x[7, k // 3] = -1000.0               # one code left
    x[8] = np.nan
    x[9, 0], x[9, k - 1] = np.inf, -np.inf
    x[10] = -np.inf
    x[10, 0] = np.nan
    x[11] = 1e4 + x[11]
    codes = rng.integers(0, k, 14)
    codes[7] = k // 3
    codes[12], codes[13] = -1, k         # none given; none of the k
    for beta in (1.0, 0.03, 20.0):
        c = Call(ctx, R.pack(x, kind), kind, beta, codes, top=3, pad=1, offset=1).check()
        c.grad(rng.standard_normal(14), rng.standard_normal(14) * 0.1)
        c.grad(rng.standard_normal(14), None)
        c.grad(None, rng.standard_normal(14))


@pytest.mark.parametrize("kind", R.TYPES)
@pytest.mark.parametrize("pad,offset", [(0, 0), (0, 1), (1, 0), (2, 3), (5, 2), (8, 0), (64, 7)])
def test_strides_and_in_place(ctx, kind, pad, offset):
    rng = np.random.default_rng([pad, offset])
    for n, k in ((9, 40), (5, 256), (3, 1001), (2, 5003), (2, 20000)):
        x = R.pack(_rows(rng, n, k), kind)
        c = Call(ctx, x, kind, 1.5, rng.integers(0, k, n), 2, 3, top=4, pad=pad, offset=offset).check()
        away = c.grad(rng.standard_normal(n), rng.standard_normal(n), pad=3)
        assert away.shape == (n, k)
        c.grad(rng.standard_normal(n), rng.standard_normal(n), inplace=True)


@pytest.mark.parametrize("n,k", [(3, 30), (2, 300), (2, 3000)])
def test_gradient_against_differences(ctx, n, k):
    """The formula's gradient against the slope of the plain form, by central differences in 64 bits: with steps of 1e-4 their
    error is about 1e-8 of the third derivative plus 1e-12 of rounding."""
    rng = np.random.default_rng([n, k, 5])
    beta, x, codes = 0.8, R.pack(_rows(rng, n, k, 1.5), "f32"), rng.integers(0, k, n)
    gl, gh = rng.standard_normal(n).astype(np.float32), rng.standard_normal(n).astype(np.float32)
    got = Call(ctx, x, "f32", beta, codes, top=0).grad(gl, gh)

    def loss(v, i):
        st = R.statistics(v[None], beta)
        return gl[i] * st["lp"][0, codes[i]] + gh[i] * st["H"][0]
    h = 1e-4
    for i in range(n):
        for j in [codes[i], int(np.argmax(x[i]))] + list(rng.integers(0, k, 20)):
            up, down = x[i].astype(np.float64), x[i].astype(np.float64)
            up[j] += h
            down[j] -= h
            slope = (loss(up, i) - loss(down, i)) / (2 * h)
            assert abs(got[i, j] - slope) < 1e-6 + 1e-5 * abs(slope)


def test_outputs_left_out(ctx):
    rng = np.random.default_rng(8)
    for n, k in ((5, 100), (2, 30000)):
        x = ctx.to_device(_rows(rng, n, k).astype(np.float32))
        codes, m = ctx.to_device(rng.integers(0, k, n).astype(np.int32)), [ctx.empty(n, np.float32) for _ in range(2)]
        tl, tc = ctx.empty((n, 3), np.float32), ctx.empty((n, 3), np.int32)
        ctx.code_logprobs("f32", x, n, k, k, 1.0, 4, None, 1, 0, None, m[0], None, None)
        assert np.array_equal(m[0].download(), x.download().max(1))
        ctx.code_logprobs("f32", x, n, k, k, 1.0, 4, None, 1, 3, None, None, None, None, tl, tc)
        assert np.array_equal(tc.download(), R.best(x.download().astype(np.float64), 3))
        ctx.code_logprobs("f32", x, n, k, k, 1.0, 4, codes, 1, 0, m[1], None, None, None)
        st = R.statistics(x.download().astype(np.float64), 1.0)
        assert np.allclose(m[1].download(), st["lp"][np.arange(n), codes.download()], atol=1e-4, rtol=0)
        ctx.code_logprobs("f32", x, n, k, k, 1.0, 4, None, 1, 0, None, None, None, None)


def test_same_call_same_bits(ctx):
    """Two runs of a call give the same bits, long rows in parts and candidates in any order included."""
    rng = np.random.default_rng(10)
    for n, k in ((3, 65536), (700, 256), (40, 9000)):
        c = Call(ctx, R.pack(_rows(rng, n, k), "bf16"), "bf16", 1.0, rng.integers(0, k, n), top=20)
        first = [o.download() for o in (*c.out, c.top_lp, c.top_code)]
        c.run()
        for a, b in zip(first, (*c.out, c.top_lp, c.top_code)):
            assert np.array_equal(a.view(np.uint32), b.download().view(np.uint32))


def test_two_contexts_and_a_run_together(ctx):
    """Trained codebook, codes of vq_assign, 8-bit scores, log probabilities, gradient: as they are used, in two contexts
    whose calls interleave."""
    import vq_amd
    from vq_amd import synth
    n, dim, k = 3000, 32, 64
    x = synth.gaussian_mixture(n, dim, 64, 0.1, seed=3)
    init, reseed = synth.index_streams(n, 1, k, 4, seed=5)
    other = vq_amd.Context(0)
    got = []
    for c in (ctx, other):
        dx, cb, codes = c.to_device(x), c.empty((1, k, dim), np.float32), c.empty((n, 1), np.uint8)
        c.lbg_fit(dx, n, dim, 1, dim, k, 4, init, reseed, cb)
        c.assign(vq_amd.SQEUCLIDEAN, dx, n, dim, 1, dim, k, cb, codes)
        book = cb.download()[0].astype(np.float64)
        xq, xs, wq, ws = c.empty((n, dim), np.int8), c.empty(n, np.float32), c.empty((k, dim), np.int8), c.empty(k, np.float32)
        bias = c.to_device((-0.5 * (book ** 2).sum(1)).astype(np.float32))
        got.append((c, dx, cb, codes, xq, xs, wq, ws, bias, c.empty((n, k), np.float32), [c.empty(n, np.float32) for _ in range(4)],
                    c.empty((n, 2), np.float32), c.empty((n, 2), np.int32), c.to_device(np.ones(n, np.float32)), c.empty((n, k), np.float32)))
    for step in range(4):
        for c, dx, cb, codes, xq, xs, wq, ws, bias, scores, outs, tl, tc, ones, grad in got:
            if step == 0:
                c.rows_i8("f32", dx, n, dim, dim, xq, dim, xs)
                c.rows_i8("f32", cb, k, dim, dim, wq, dim, ws)
            elif step == 1:
                c.scores_i8(xq, xs, n, dim, wq, ws, k, dim, dim, bias, "f32", scores, k)
            elif step == 2:
                c.code_logprobs("f32", scores, n, k, k, 10.0, 1, codes, 1, 2, *outs, tl, tc)
            else:
                c.code_logprobs_grad("f32", scores, n, k, k, 10.0, 1, codes, 1, *outs[1:], ones, None, grad, k)
    for c, dx, cb, codes, xq, xs, wq, ws, bias, scores, outs, tl, tc, ones, grad in got:
        q, s = R.rows_i8(x.astype(np.float64))
        assert np.array_equal(xq.download(), q) and np.array_equal(xs.download(), s)
        q2, s2 = R.rows_i8(cb.download()[0].astype(np.float64))
        want, tol = R.scores(q, s, q2, s2, bias.download(), "f32")
        sc = scores.download()
        assert (np.abs(sc - want) <= tol).all()
        st = R.statistics(sc.astype(np.float64), 10.0)
        tL, tH = R.bounds(st, k)
        lp, m, L, H = (o.download() for o in outs)
        assert (np.abs(L - st["L"]) <= tL).all() and (np.abs(H - st["H"]) <= tH).all()
        assert np.array_equal(tc.download(), R.best(sc.astype(np.float64), 2))
        assert (tc.download()[:, 0] == codes.download()[:, 0]).mean() > 0.9  # the nearest codeword is the likeliest, nearly always
        g, err = R.grad(sc.astype(np.float64), 10.0, codes.download()[:, 0].astype(np.int64), m, L, H, np.ones(n), None)
        assert (np.abs(grad.download() - g) <= err + R.U24 * np.abs(g)).all()
    other.close()


def test_graph(ctx):
    """The four calls captured on the context's stream, replayed several times with other work between."""
    import vq_amd
    hip = C.CDLL("libamdhip64.so")
    lib = vq_amd._ffi.lib()
    stream = C.c_void_p(lib.vq_ctx_stream(ctx._h))
    rng = np.random.default_rng(12)
    n, dim, k = 3, 200, 40000
    rows, w = ctx.to_device(rng.standard_normal((n, dim)).astype(np.float32)), ctx.to_device(rng.integers(-127, 128, (k, dim)).astype(np.int8))
    xq, xs, ws = ctx.empty((n, dim), np.int8), ctx.empty(n, np.float32), ctx.to_device(rng.uniform(0.001, 0.01, k).astype(np.float32))
    scores, codes = ctx.empty((n, k), np.float32), ctx.to_device(rng.integers(0, k, n).astype(np.int32))
    outs, tl, tc = [ctx.empty(n, np.float32) for _ in range(4)], ctx.empty((n, 9), np.float32), ctx.empty((n, 9), np.int32)
    ones, grad = ctx.to_device(np.ones(n, np.float32)), ctx.empty((n, k), np.float32)

    def calls(c):
        c.rows_i8("f32", rows, n, dim, dim, xq, dim, xs)
        c.scores_i8(xq, xs, n, dim, w, ws, k, dim, dim, None, "f32", scores, k)
        c.code_logprobs("f32", scores, n, k, k, 1.0, 4, codes, 1, 9, *outs, tl, tc)
        c.code_logprobs_grad("f32", scores, n, k, k, 1.0, 4, codes, 1, *outs[1:], ones, ones, grad, k)

    calls(ctx)
    ctx.sync()
    graph, run = C.c_void_p(), C.c_void_p()
    assert hip.hipStreamBeginCapture(stream, 2) == 0
    calls(ctx)
    assert hip.hipStreamEndCapture(stream, C.byref(graph)) == 0
    assert hip.hipGraphInstantiate(C.byref(run), graph, None, None, 0) == 0
    for rep in range(4):
        rows.upload(rng.standard_normal((n, dim)).astype(np.float32))
        assert hip.hipGraphLaunch(run, stream) == 0
        ctx.sync()
        got = [a.download() for a in (xq, xs, scores, *outs, tl, tc, grad)]
        # eager work between the replays, a larger size among it
        big = Call(ctx, R.pack(_rows(rng, 2, 70000 + 50000 * rep), "f32"), "f32", 1.0, np.zeros(2, np.int64), top=32)
        big.check()
        calls(ctx)
        ctx.sync()
        for a, b in zip(got, (xq, xs, scores, *outs, tl, tc, grad)):
            assert np.array_equal(a.view(np.uint8), b.download().view(np.uint8))
    assert hip.hipGraphExecDestroy(run) == 0 and hip.hipGraphDestroy(graph) == 0


def test_capture_before_the_workspace_is_there():
    """A call whose workspace would have to grow is refused while the stream is captured; the capture goes on with a call
    that needs none, and the refused call runs afterwards."""
    import vq_amd
    hip, lib = C.CDLL("libamdhip64.so"), vq_amd._ffi.lib()
    c = vq_amd.Context(0)
    stream = C.c_void_p(lib.vq_ctx_stream(c._h))
    x, lp = c.to_device(np.linspace(0, 5, 70000, dtype=np.float32)), c.empty(2, np.float32)
    codes = c.to_device(np.full(1, 7, np.int32))
    graph, run = C.c_void_p(), C.c_void_p()
    assert hip.hipStreamBeginCapture(stream, 2) == 0
    with pytest.raises(vq_amd.VqError) as e:
        c.code_logprobs("f32", x, 1, 70000, 70000, 1.0, 4, codes, 1, 0, lp, None, None, None)
    assert e.value.code == vq_amd._ffi.ERR_UNSUPPORTED and "capture" in str(e.value)
    c.code_logprobs("f32", x, 1, 70000, 100, 1.0, 4, codes, 1, 0, lp, None, None, None)
    assert hip.hipStreamEndCapture(stream, C.byref(graph)) == 0
    assert hip.hipGraphInstantiate(C.byref(run), graph, None, None, 0) == 0
    for _ in range(3):
        assert hip.hipGraphLaunch(run, stream) == 0
        c.sync()
        st = R.statistics(x.download()[None, :100].astype(np.float64), 1.0)
        assert abs(lp.download()[0] - st["lp"][0, 7]) < 1e-5
        c.code_logprobs("f32", x, 1, 70000, 70000, 1.0, 4, codes, 1, 0, lp, None, None, None)
        st = R.statistics(x.download()[None].astype(np.float64), 1.0)
        assert abs(lp.download()[0] - st["lp"][0, 7]) < 1e-4
    assert hip.hipGraphExecDestroy(run) == 0 and hip.hipGraphDestroy(graph) == 0
    c.close()


def test_refusals_leave_the_context_usable(ctx):
    import vq_amd
    x, codes, lp = ctx.to_device(np.zeros((2, 8), np.float32)), ctx.to_device(np.zeros(2, np.int32)), ctx.empty(2, np.float32)
    for change in (dict(k=9), dict(beta=0.0), dict(top=33), dict(cb=3)):
        a = {**dict(k=8, beta=1.0, cb=4, top=0), **change}
        with pytest.raises(vq_amd.VqError) as e:
            ctx.code_logprobs("f32", x, 2, 8, a["k"], a["beta"], a["cb"], codes, 1, a["top"], lp, None, None, None, lp, lp)
        assert e.value.code in (vq_amd._ffi.ERR_INVALID_ARG, vq_amd._ffi.ERR_UNSUPPORTED) and "Invalid parameter" in str(e.value)
    with pytest.raises(vq_amd.VqError):
        ctx.code_logprobs_grad("f32", x, 2, 8, 8, 1.0, 4, codes, 1, lp, lp, None, None, None, x, 8)
    ctx.code_logprobs("f32", x, 2, 8, 8, 1.0, 4, codes, 1, 0, lp, None, None, None)
    assert np.allclose(lp.download(), -np.log(8), atol=1e-6)
