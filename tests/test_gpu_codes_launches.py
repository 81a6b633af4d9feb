"""GPU: calls of models over codes that take more launches than one by the size of a grid alone."""
import numpy as np
import pytest

import codes_ref as Q
from test_gpu_embed import near

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    import vq_amd
    c = vq_amd.Context(0)
    yield c
    c.close()


@pytest.mark.parametrize("rest", [False, True])
def test_gradients_of_more_rows_than_a_launch_takes(ctx, rest):
    """2^22 rows of a gradient's own call are a launch's."""
    n, k, period = (1 << 22) + 6, 8, 7
    i = np.arange(n) % period
    few = (np.arange(period)[:, None] * 0.25 * np.arange(k)).astype(np.float32)
    lp, code = np.log(np.array([[0.5, 0.2]], np.float32)).repeat(period, 0), np.stack([np.arange(period), (np.arange(period) + 3) % k], 1).astype(np.int32)
    g = (1.0 + np.arange(period)).astype(np.float32)
    dx, dl, dc, dg = (ctx.to_device(np.ascontiguousarray(a[i])) for a in (few, lp, code, g))
    out = [ctx.empty(n, np.float32) for _ in range(4)]
    grad = ctx.empty((n, k), np.float32)
    ctx.code_distill("f32", dx, n, k, k, 1.0, 2, dl, dc, 2, rest, *out)
    ctx.code_distill_grad("f32", dx, n, k, k, 1.0, 2, dl, dc, 2, rest, *out[1:], dg, grad, k)
    m, L, lr = (o.download() for o in out[1:])
    y = grad.download()
    want, err = Q.distill_grad(few.astype(np.float64), 1.0, lp, code, rest, m[:period], L[:period], lr[:period], g)
    near(y[:period].astype(np.float64), want, Q.rounded(want, err, "f32"))
    for r in range(period):  # the same rows, the same bits
        for a in (m, L, lr, y):
            assert (a[r::period] == a[r]).all()


def test_columns_of_a_gradient_in_two_launches(ctx):
    """Rows of the widest table: 513 groups of its codes times 16,384 groups of columns are more workgroups than a launch takes, so the last columns
    go in a second one.  Added to what is there, so that the rows that nobody names, of 138 GB in all, are not touched."""
    import vq_amd
    k, dim, n = 65_600, 1 << 20, 9
    try:
        grad = ctx.empty((k * dim,), np.float16)
    except vq_amd.VqError as e:
        pytest.skip(f"no memory for the table's gradient: {e}")
    try:
        lib, row = vq_amd._ffi.lib(), 2 * dim
        rng = np.random.default_rng(0)
        g = rng.standard_normal((n, dim)).astype(np.float32)
        codes = np.array([0, 5, k - 1, 5, 40_000, -1, 5, k, 0], np.int32)
        old = rng.standard_normal(dim).astype(np.float16)
        named = [0, 5, 40_000, k - 1]
        put = lambda c: ctx._check(lib.vq_h2d(ctx._h, grad.ptr + c * row, old.ctypes.data, row))
        beside = [1, 4, 6, k - 2]
        for c in named + beside:
            put(c)
        ctx.code_embed_grad("f32", ctx.to_device(g), n, dim, dim, 1, 4, ctx.to_device(codes), 1, 0.5, k, True, "f16", grad, dim)
        for c in named + beside:
            got = np.empty(dim, np.float16)
            ctx._check(lib.vq_d2h(ctx._h, got.ctypes.data, grad.ptr + c * row, row))
            rows = g[codes == c].astype(np.float64)
            want = old + 0.5 * rows.sum(axis=0)
            if c in beside:
                assert np.array_equal(got, old)
            # three sums and a product in f32, rounded to f16
            near(got.astype(np.float64), want, Q.rounded(want, 5 * 2.0 ** -24 * (np.abs(old) + np.abs(rows).sum(axis=0)), "f16"))
    finally:
        grad.free()


def test_a_graph_of_rows_in_parts_with_their_gradient(ctx):
    """Loss and gradient of fewer than 64 long rows, whose sums go from launch to launch through the context's buffer: captured, replayed between eager
    calls of other sizes, every replay against the eager result."""
    from test_gpu_scores_workspace import Captured
    rng = np.random.default_rng(7)
    n, k, top = 9, 40_003, 6
    x = rng.standard_normal((n, k)).astype(np.float32)
    lp, code = np.log(np.full((n, top), 0.15, np.float32)), np.stack([rng.permutation(k)[:top] for _ in range(n)]).astype(np.int32)
    dx, dl, dc, dg = (ctx.to_device(a) for a in (x, lp, code, rng.random(n).astype(np.float32)))
    out, grad = [ctx.empty(n, np.float32) for _ in range(4)], ctx.empty((n, k), np.float32)
    call = lambda rows=n: ctx.code_distill("f32", dx, rows, k, k, 1.0, top, dl, dc, top, True, *out, dg, grad, k)
    call()
    ctx.sync()
    graph = Captured(ctx, call)
    for rep in range(4):
        dx.upload(rng.standard_normal((n, k)).astype(np.float32) * (rep + 1))
        grad.upload(np.zeros((n, k), np.float32))
        graph.launch()
        got = [a.download() for a in (*out, grad)]
        call(3 + rep)
        call()
        ctx.sync()
        for a, b in zip(got, (*out, grad)):
            assert np.array_equal(a, b.download())
