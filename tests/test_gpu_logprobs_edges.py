"""GPU: log probabilities of codes and their gradient at the edges of what the header promises, for every way a row goes
through the GPU, against plain forms in 64 bits (scores_ref.py)."""
import numpy as np
import pytest

import scores_ref as R
from test_gpu_logprobs import Call, _rows

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    import vq_amd
    c = vq_amd.Context(0)
    yield c
    c.close()


# rows of a lane (below a vector of 16 bytes, and not), of 4 and 8 lanes, of a wave, of a workgroup, in parts
LENGTHS = [2, 3, 6, 12, 40, 200, 300, 900, 3000, 6000, 20000, 50001]


@pytest.mark.parametrize("kind", R.TYPES)
@pytest.mark.parametrize("k", LENGTHS)
def test_gradient_of_rows_without_a_code_that_can_be(ctx, kind, k):
    """A row of -inf only has gradient zero, a code of k or above among them; such a code makes any other row's gradient NaN."""
    rng = np.random.default_rng(k)
    x = _rows(rng, 6, k)
    x[1], x[2], x[4] = -np.inf, -np.inf, -np.inf
    c = Call(ctx, R.pack(x, kind), kind, 1.0, np.array([0, k, k - 1, k, -1, k + 100]), top=2).check()
    got = c.grad(rng.standard_normal(6), rng.standard_normal(6))
    assert (got[[1, 2, 4]] == 0).all() and np.isnan(got[[3, 5]]).all() and np.isfinite(got[0]).all()
    c.grad(rng.standard_normal(6), None)


@pytest.mark.parametrize("kind", R.TYPES)
@pytest.mark.parametrize("k", [1] + LENGTHS)
def test_no_probability_above_one(ctx, kind, k):
    """Rows that one code decides, at scores of many sizes: no log probability is above zero, no entropy and no L below."""
    rng = np.random.default_rng(k)
    n = 400 if k < 5000 else 60
    x = rng.uniform(-30, 30, (n, 1)) * 2.0 ** rng.integers(-3, 6, (n, 1)) - 2000.0 * rng.integers(1, 4, (n, k))
    best = rng.integers(0, k, n)
    x[np.arange(n), best] = rng.uniform(-30, 30, n) * 2.0 ** rng.integers(-3, 6, n)
    for beta in (1.0, 0.375, 11.0):
        c = Call(ctx, R.pack(x, kind), kind, beta, best, top=2).check()
        lp, m, L, H = (o.download()[:n] for o in c.out)
        assert (lp <= 0).all(), (lp.max(), (lp > 0).sum())
        assert (L >= 0).all() and (H >= 0).all(), (L.min(), H.min())
        assert (c.top_lp.download()[:n] <= 0).all()
        with np.errstate(divide="ignore"):
            assert not np.isnan(np.log1p(-np.exp(lp))).any()


@pytest.mark.parametrize("kind", R.TYPES)
@pytest.mark.parametrize("k", [2, 6, 12, 40, 100, 250])
def test_a_row_does_not_depend_on_its_neighbours(ctx, kind, k):
    """Rows of several to a wave: the same bits whatever scores the other rows hold."""
    rng = np.random.default_rng(k)
    n = 192
    x = _rows(rng, n, k, 8.0) + rng.uniform(-300, 300, (n, 1))
    codes = rng.integers(0, k, n)

    def outputs(v):
        c = Call(ctx, R.pack(v, kind), kind, 0.875, codes, top=2).check()
        return [o.download()[:n] for o in (*c.out, c.top_lp, c.top_code)]
    first = outputs(x)
    for far in (3e4, 6e4 if kind == "f16" else 5e6, -6e4 if kind == "f16" else 3e38, -np.inf, np.nan):
        y = x.copy()
        y[1::2] = y[1::2] * 0.01 + far if abs(far) < 1e30 else far
        for a, b in zip(first, outputs(y)):
            assert np.array_equal(a[::2].view(np.uint32), b[::2].view(np.uint32))


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("k", LENGTHS[1:])
def test_scores_further_apart_than_a_number(ctx, kind, k):
    """Scores whose difference is beyond binary32: their log probability, beta times it, is within for a beta below 1."""
    rng = np.random.default_rng(k)
    x = np.full((5, k), -np.inf)
    x[:, 0], x[:, k - 1] = 3e38, -3e38
    x[1, k // 2] = -2.5e38
    x[2] = rng.uniform(-3e38, 3e38, k)
    x[2, 0], x[2, k - 1] = 3.3e38, -3.3e38
    x[3, 0] = 1.0
    x[4, k // 2] = 3e38
    for beta in (0.5, 2.0 ** -10, 2.0 ** -60, 2.0 ** -99, 3.0):
        c = Call(ctx, R.pack(x, kind), kind, beta, np.array([k - 1, k - 1, k - 1, k - 1, k - 1]), top=4).check()
        lp = c.out[0].download()[:5]
        assert np.isfinite(lp).all() or beta == 3.0
        c.grad(rng.standard_normal(5), rng.standard_normal(5))


@pytest.mark.parametrize("kind", R.TYPES)
@pytest.mark.parametrize("k", LENGTHS)
def test_gradient_where_the_probability_is_zero(ctx, kind, k):
    """Zero there, but for the code's own term, whatever the loss's gradients are, infinities among them."""
    rng = np.random.default_rng(k)
    n = 6
    x = _rows(rng, n, k)
    gone = rng.random((n, k)) < 0.5
    gone[:, 0], gone[:, k - 1] = False, True
    x[gone] = -np.inf
    gl, gh = rng.standard_normal(n), rng.standard_normal(n)
    gl[1], gl[2], gh[3], gh[4] = np.inf, -np.inf, 3e38, -np.inf
    codes = np.array([0, 0, -1, 0, 0, k - 1])
    c = Call(ctx, R.pack(x, kind), kind, 2.0, codes, top=1).check()
    dgl, dgh = ctx.to_device(gl.astype(np.float32)), ctx.to_device(gh.astype(np.float32))
    out = ctx.to_device(R.pack(np.full((n, k), 5.0), kind))
    ctx.code_logprobs_grad(kind, c.ptr, n, k, k, 2.0, 4, c.dcodes, 1, c.out[1], c.out[2], c.out[3], dgl, dgh, out, k)
    got = R.unpack(out.download(), kind)
    own = np.zeros((n, k), bool)
    own[5, k - 1] = True
    assert (got[gone & ~own] == 0).all()
    want = 2.0 * np.float64(np.float32(gl[5]))
    assert abs(got[5, k - 1] - want) <= (R.HALF_STEP[kind] + R.U24) * 1.01 * abs(want)
    assert not np.isfinite(got[1, 0]) and np.isfinite(got[0]).all()
