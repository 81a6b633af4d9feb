"""GPU: 8-bit scores and log probabilities of more rows than one launch takes: the rows on both sides of the border, and what
belongs to them, lie where they should.  The rows repeat with a period that divides no launch, so that few of them are
computed in 64 bits (scores_ref.py)."""
import numpy as np
import pytest

import scores_ref as R

pytestmark = pytest.mark.gpu
PERIOD = 997
ROWS = 1 << 23  # of a launch of rows to 8 bits, and of gradients


@pytest.fixture(scope="module")
def ctx():
    import vq_amd
    c = vq_amd.Context(0)
    yield c
    c.close()


def _repeated(a, n):
    return np.concatenate([a] * (n // len(a)) + [a[:n % len(a)]])


def _checked(got, want, near):
    """got: n rows; want: PERIOD of them; near(got, want, at): whether they agree, `at` the rows of the period."""
    for lo in range(0, len(got), PERIOD):
        part = got[lo:lo + PERIOD]
        if not (lo and np.array_equal(part.view(np.uint8), got[:len(part)].view(np.uint8))):  # (the same bits as the first ones)
            assert near(part, want[:len(part)], slice(0, len(part))).all(), lo


@pytest.mark.parametrize("dim", [3, 16])
def test_rows(ctx, dim):
    n, ld, ld_q = ROWS + 1500, dim + 1, dim + 3
    x = np.random.default_rng(dim).standard_normal((PERIOD, ld)) * 3
    x = R.pack(x, "f16")
    dq, ds = ctx.to_device(np.full((n, ld_q), 99, np.int8)), ctx.empty(n, np.float32)
    ctx.rows_i8("f16", ctx.to_device(_repeated(x, n)), n, ld, dim, dq, ld_q, ds)
    q, s = R.rows_i8(R.unpack(x[:, :dim], "f16"))
    got = dq.download()
    assert (got[:, dim:] == 99).all()
    assert np.array_equal(got[:, :dim], _repeated(q, n)) and np.array_equal(ds.download(), _repeated(s, n))


@pytest.mark.parametrize("k", [3, 16])
def test_gradients(ctx, k):
    n, ld = ROWS + 1500, k + 1
    rng = np.random.default_rng(k)
    x = R.pack(rng.standard_normal((PERIOD, ld)), "f16")
    codes = rng.integers(-1, k + 1, (PERIOD, 2)).astype(np.int32)
    gl, gh = rng.standard_normal(PERIOD).astype(np.float32), rng.standard_normal(PERIOD).astype(np.float32)
    dx, dc, dgl, dgh = (ctx.to_device(_repeated(a, n)) for a in (x, codes, gl, gh))
    lp, m, L, H = (ctx.empty(n, np.float32) for _ in range(4))
    ctx.code_logprobs("f16", dx, n, ld, k, 1.5, 4, dc, 2, 0, lp, m, L, H)
    out = ctx.to_device(np.full((n, k + 2), 9, np.float16))
    ctx.code_logprobs_grad("f16", dx, n, ld, k, 1.5, 4, dc, 2, m, L, H, dgl, dgh, out, k + 2)
    hm, hL, hH = (a.download()[:PERIOD] for a in (m, L, H))
    want, err = R.grad(R.unpack(x[:, :k], "f16"), 1.5, codes[:, 0].astype(np.int64), hm, hL, hH, gl, gh)
    tol = err + 1.01 * R.HALF_STEP["f16"] * (np.abs(want) + err) + R.LEAST["f16"]
    got = out.download()
    assert (got[:, k:] == 9).all()

    def near(a, b, at):
        return (np.abs(a.astype(np.float64) - b) <= tol[at]) | (np.isnan(a) & np.isnan(b))
    _checked(np.ascontiguousarray(got[:, :k]), want, near)


def test_parts_of_many_rows(ctx):
    """Two parts per row and 32 alternatives: 125,203 rows fill the 64 MiB of a launch's parts."""
    n, k, top, ld, stride = 125_203 + 400, 16_385, 32, 16_387, 3
    rng = np.random.default_rng(1)
    x = rng.standard_normal((PERIOD, ld)).astype(np.float32)
    x[5], x[17, 16_384], x[90] = -np.inf, 9.0, 1.0
    x = R.pack(x, "bf16")
    codes = rng.integers(-1, k + 1, (PERIOD, stride)).astype(np.int32)
    dx, dc = ctx.to_device(_repeated(x, n)), ctx.to_device(_repeated(codes, n))
    out = [ctx.to_device(np.full(n + 1, 7, np.float32)) for _ in range(4)]
    tl, tc = ctx.to_device(np.full((n + 1, top), 7, np.float32)), ctx.to_device(np.full((n + 1, top), 7, np.int32))
    ctx.code_logprobs("bf16", dx, n, ld, k, 1.0, 4, dc, stride, top, *out, tl, tc)
    v = R.unpack(x[:, :k], "bf16")
    st = R.statistics(v, 1.0)
    tL, tH = R.bounds(st, k)
    c = codes[:, 0].astype(np.int64)
    at = np.clip(c, 0, k - 1)
    rows = np.arange(PERIOD)
    lp = np.where(c < 0, 0.0, np.where(c >= k, np.nan, st["lp"][rows, at]))
    tlp = (2 * np.abs(st["d"][rows, at]) + np.abs(st["lp"][rows, at])) * R.U24 * 1.01 + tL
    for o, want, tol in zip(out, (lp, st["m"], st["L"], st["H"]), (tlp, 0 * tL, tL, tH)):
        got = o.download()
        assert got[n] == 7
        with np.errstate(invalid="ignore"):
            _checked(got[:n], want, lambda a, b, i: (a == b) | (np.abs(a - b) <= tol[i]) | (np.isnan(a) & np.isnan(b)))
    got = tc.download()
    assert (got[n] == 7).all()
    best = R.best(v, top)
    _checked(got[:n], best, lambda a, b, i: a == b)
    got = tl.download()
    assert (got[n] == 7).all()
    j = np.clip(best, 0, k - 1)
    want = np.where(best < 0, -np.inf, np.take_along_axis(st["lp"], j, 1))
    with np.errstate(invalid="ignore"):
        tol = (2 * np.abs(np.take_along_axis(st["d"], j, 1)) + np.abs(want)) * R.U24 * 1.01 + tL[:, None]
        _checked(got[:n], want, lambda a, b, i: (a == b) | (np.abs(a - b) <= tol[i]))


@pytest.mark.parametrize("pad", [0, 1])
def test_copied_rows(ctx, pad):
    """Rows of 131,071 components are copied 4096 at a time."""
    n, dim, k = 4096 * 2 + 77, 131_071, 33
    ld, ldw = dim + 2 * pad, (dim + 15) // 16 * 16 if pad else dim
    rng = np.random.default_rng(pad)
    x, w = rng.integers(-127, 128, (PERIOD, ld)).astype(np.int8), rng.integers(-127, 128, (k, ldw)).astype(np.int8)
    xs, ws = rng.uniform(0.001, 0.01, PERIOD).astype(np.float32), rng.uniform(0.001, 0.01, k).astype(np.float32)
    bias = rng.standard_normal(k).astype(np.float32)
    out = ctx.to_device(np.full((n + 1, k + 1), -3, np.float32))
    ctx.scores_i8(ctx.to_device(_repeated(x, n)), ctx.to_device(_repeated(xs, n)), n, ld, ctx.to_device(w), ctx.to_device(ws), k, ldw, dim,
                  ctx.to_device(bias), "f32", out, k + 1)
    got = out.download()
    assert (got[n] == -3).all() and (got[:, k:] == -3).all()
    want, tol = R.scores(x[:, :dim], xs, w[:, :dim], ws, bias, "f32")
    _checked(np.ascontiguousarray(got[:n, :k]), want, lambda a, b, at: np.abs(a - b) <= tol[at])


@pytest.mark.parametrize("aligned", [False, True])
def test_launches_of_scores(ctx, aligned):
    """64 x 65,535 rows are a launch of few codes."""
    n, dim, k = 65_535 * 64 + 1500, 16, 5
    ld = 16 if aligned else 17
    rng = np.random.default_rng(3)
    x, w = rng.integers(-127, 128, (PERIOD, ld)).astype(np.int8), rng.integers(-127, 128, (k, 16)).astype(np.int8)
    xs, ws = rng.uniform(0.5, 1, PERIOD).astype(np.float32), rng.uniform(0.5, 1, k).astype(np.float32)
    out = ctx.to_device(np.full((n + 1, k + 1), -3, np.float16))
    ctx.scores_i8(ctx.to_device(_repeated(x, n)), ctx.to_device(_repeated(xs, n)), n, ld, ctx.to_device(w), ctx.to_device(ws), k, 16, dim, None, "f16", out, k + 1)
    got = out.download()
    assert (got[n] == -3).all() and (got[:, k:] == -3).all()
    want, tol = R.scores(x[:, :dim], xs, w, ws, None, "f16")
    assert np.abs(want).max() < 65_000
    _checked(np.ascontiguousarray(got[:n, :k]), want, lambda a, b, at: np.abs(a - b) <= tol[at])
