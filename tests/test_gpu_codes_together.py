"""GPU: the operators of models over codes one after another, as a training step and a server use them, beside the calls that were there; in
captured graphs; from two contexts at once."""
import ctypes as C

import numpy as np
import pytest

import codes_ref as Q
import scores_ref as R
from test_gpu_embed import near
from test_gpu_scores_workspace import Captured

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    import vq_amd
    c = vq_amd.Context(0)
    yield c
    c.close()


def test_a_training_step(ctx):
    """Codes of four stages to rows, rows to 8-bit scores, a teacher's alternatives from its own scores, loss and gradient against
    them in place, the gradient of the rows (on the host) and of the tables; each against its plain form on what the one before left."""
    rng = np.random.default_rng(0)
    n, m, k, dim, answers, top = 300, 4, 500, 96, 2000, 8
    codes = rng.integers(-1, k, (n, m)).astype(np.int32)
    table = rng.standard_normal((m * k, dim)).astype(np.float32)
    rows = ctx.empty((n, dim), np.float32)
    dt, dc = ctx.to_device(table), ctx.to_device(codes)
    ctx.code_embed("f32", dt, k, dim, dim, m, 4, dc, n, m, 0.5, "f32", rows, dim)
    x = rows.download()
    want, err = Q.embed(table.reshape(m, k, dim).astype(np.float64), codes, 0.5)
    near(x.astype(np.float64), want, Q.rounded(want, err, "f32"))
    q, qs, w, ws = ctx.empty((n, dim), np.int8), ctx.empty(n, np.float32), rng.integers(-127, 128, (answers, dim)).astype(np.int8), np.full(answers, 0.002, np.float32)
    dw, dws, scores = ctx.to_device(w), ctx.to_device(ws), ctx.empty((n, answers), np.float32)
    ctx.rows_i8("f32", rows, n, dim, dim, q, dim, qs)
    ctx.scores_i8(q, qs, n, dim, dw, dws, answers, dim, dim, None, "f32", scores, answers)
    s = scores.download()
    # the teacher: other scores, its best answers
    z = (s + rng.standard_normal(s.shape)).astype(np.float32)
    dz, tl, tc = ctx.to_device(z), ctx.empty((n, top), np.float32), ctx.empty((n, top), np.int32)
    ctx.code_logprobs("f32", dz, n, answers, answers, 1.0, 4, None, 1, top, None, None, None, None, tl, tc)
    loss, mx, L, lr = (ctx.empty(n, np.float32) for _ in range(4))
    g = rng.random(n).astype(np.float32)
    dg = ctx.to_device(g)
    ctx.code_distill("f32", scores, n, answers, answers, 1.0, top, tl, tc, top, True, loss, mx, L, lr, dg, scores, answers)
    lp, code = tl.download(), tc.download()
    o = Q.distill(s.astype(np.float64), 1.0, lp, code, True)
    near(loss.download().astype(np.float64), o["loss"], o["tloss"])
    y = scores.download()
    wy, err = Q.distill_grad(s.astype(np.float64), 1.0, lp, code, True, mx.download(), L.download(), lr.download(), g)
    near(y.astype(np.float64), wy, Q.rounded(wy, err, "f32"))
    down = (y @ (w * ws[:, None])).astype(np.float32)
    grad = ctx.to_device(np.ones((m * k, dim), np.float32))
    ctx.code_embed_grad("f32", ctx.to_device(down), n, dim, dim, m, 4, dc, m, 0.5, k, True, "f32", grad, dim)
    want, err = Q.embed_grad(down.astype(np.float64), codes, 0.5, k, np.ones((m, k, dim)))
    near(grad.download().astype(np.float64).reshape(m, k, dim), want, Q.rounded(want, err, "f32"))


def test_a_step_of_a_server(ctx):
    """Drafts verified, and the codes that come out looked up as they are: none behind the next one."""
    rng = np.random.default_rng(1)
    n, draft, k, dim = 20, 3, 700, 40
    t = R.unpack(R.pack(rng.standard_normal((n, draft + 1, k)) * 2, "bf16"), "bf16")
    d = R.unpack(R.pack(t[:, :draft] + 0.5 * rng.standard_normal((n, draft, k)), "bf16"), "bf16")
    codes = (d + rng.gumbel(size=d.shape)).argmax(axis=2).astype(np.int32)
    u = rng.random((n, draft + 1)).astype(np.float32)
    dt, dd = ctx.to_device(R.pack(t.reshape(-1, k), "bf16")), ctx.to_device(R.pack(d.reshape(-1, k), "bf16"))
    accepted, out = ctx.empty(n, np.int32), ctx.empty((n, draft + 1), np.int32)
    dcodes, du = ctx.to_device(codes), ctx.to_device(u)
    ctx.code_verify("bf16", dt, k, 1.0, dd, k, 1.0, n, draft, k, 4, dcodes, draft, du, draft + 1, accepted, out, draft + 1)
    table = rng.standard_normal((k, dim)).astype(np.float32)
    rows = ctx.empty((n * (draft + 1), dim), np.float32)
    ctx.code_embed("f32", ctx.to_device(table), k, dim, dim, 1, 4, out, n * (draft + 1), 1, 1.0, "f32", rows, dim)
    wa, wo = Q.verify(t, 1.0, d, 1.0, codes, u.astype(np.float64))
    assert np.array_equal(out.download(), wo) and np.array_equal(accepted.download(), wa)
    flat = wo.reshape(-1)
    assert np.array_equal(rows.download(), np.where(flat[:, None] >= 0, table[flat], np.float32(0)))


class Everything:
    """Every call at one size, on buffers of its own."""

    def __init__(self, ctx, rng, n=70, k=20001, dim=72, draft=3, positions=3000):
        self.ctx, self.n, self.k, self.dim, self.draft, self.positions = ctx, n, k, dim, draft, positions
        up = ctx.to_device
        self.scores = up(R.pack(rng.standard_normal((n, k)) * 2, "f16"))
        self.z = up(R.pack(rng.standard_normal((n, k)) * 2, "f16"))
        self.tl, self.tc = ctx.empty((n, 6), np.float32), ctx.empty((n, 6), np.int32)
        self.g = up(rng.random(n).astype(np.float32))
        self.stats = [ctx.empty(n, np.float32) for _ in range(4)]
        self.grad, self.grad2 = up(R.pack(np.zeros((n, k)), "f16")), up(R.pack(np.zeros((n, k)), "f16"))
        self.table = up(R.pack(rng.standard_normal((500, dim)), "bf16"))
        self.codes = up(rng.integers(0, 3, positions).astype(np.int32) * rng.integers(0, 166, positions).astype(np.int32))
        self.rows, self.table_grad = up(R.pack(np.zeros((positions, dim)), "bf16")), ctx.empty((500, dim), np.float32)
        seq = n // (draft + 1)
        self.seq = seq
        self.drafted = up(rng.integers(0, k, (seq, draft)).astype(np.int32))
        self.u = up((rng.random((seq, draft + 1)) * 0.5).astype(np.float32))
        self.accepted, self.out = ctx.empty(seq, np.int32), ctx.empty((seq, draft + 1), np.int32)

    def calls(self):
        c, n, k = self.ctx, self.n, self.k
        c.code_logprobs("f16", self.z, n, k, k, 1.0, 4, None, 1, 6, None, None, None, None, self.tl, self.tc)
        c.code_distill("f16", self.scores, n, k, k, 1.0, 6, self.tl, self.tc, 6, True, *self.stats, self.g, self.grad, k)
        c.code_distill("f16", self.scores, n, k, k, 1.0, 6, self.tl, self.tc, 6, True, *self.stats)
        c.code_distill_grad("f16", self.scores, n, k, k, 1.0, 6, self.tl, self.tc, 6, True, *self.stats[1:], self.g, self.grad2, k)
        c.code_embed("bf16", self.table, 500, self.dim, self.dim, 1, 4, self.codes, self.positions, 1, 2.0, "bf16", self.rows, self.dim)
        c.code_embed_grad("bf16", self.rows, self.positions, self.dim, self.dim, 1, 4, self.codes, 1, 2.0, 500, False, "f32", self.table_grad, self.dim)
        c.code_verify("f16", self.scores, k, 1.0, self.z, k, 1.0, self.seq, self.draft, k, 4, self.drafted, self.draft, self.u, self.draft + 1,
                      self.accepted, self.out, self.draft + 1)

    def results(self):
        return [a.download().view(np.uint8) for a in (*self.stats, self.grad, self.grad2, self.rows, self.table_grad, self.accepted, self.out)]


def test_capture_and_replay():
    """All calls in a graph, replayed between eager work of the context, larger calls among it; every replay against the eager results."""
    import vq_amd
    ctx = vq_amd.Context(0)
    rng = np.random.default_rng(3)
    e = Everything(ctx, rng)
    e.calls()
    ctx.sync()
    graph = Captured(ctx, e.calls)
    for rep in range(4):
        e.scores.upload(R.pack(rng.standard_normal((e.n, e.k)) * 2, "f16"))
        e.codes.upload(rng.integers(0, 500, e.positions).astype(np.int32))
        graph.launch()
        got = e.results()
        big = Everything(ctx, rng, n=40 + 40 * rep, k=60000 + 10000 * rep, positions=40000 + 5000 * rep)  # the buffer grows; the graph keeps its own
        big.calls()
        e.calls()
        ctx.sync()
        for a, b in zip(got, e.results()):
            assert np.array_equal(a, b)
        del big
    graph.close()
    ctx.close()


def test_a_capture_needs_the_workspace():
    """Calls whose buffer would have to grow are refused while the stream is captured, the capture goes on, and they run afterwards."""
    import vq_amd
    ctx = vq_amd.Context(0)
    rng = np.random.default_rng(4)
    e = Everything(ctx, rng)
    ctx.code_logprobs("f16", e.z, e.n, e.k, e.k, 1.0, 4, None, 1, 6, None, None, None, None, e.tl, e.tc)
    ctx.sync()

    def refused():
        for call in (lambda: ctx.code_embed_grad("bf16", e.rows, e.positions, e.dim, e.dim, 1, 4, e.codes, 1, 2.0, 500, False, "f32", e.table_grad, e.dim),
                     lambda: ctx.code_distill("f16", e.scores, e.n, e.k, e.k, 1.0, 6, e.tl, e.tc, 6, True, *e.stats),
                     lambda: ctx.code_verify("f16", e.scores, e.k, 1.0, e.z, e.k, 1.0, e.seq, e.draft, e.k, 4, e.drafted, e.draft, e.u, e.draft + 1,
                                             e.accepted, e.out, e.draft + 1)):
            with pytest.raises(vq_amd.VqError) as err:
                call()
            assert err.value.code == vq_amd._ffi.ERR_UNSUPPORTED and "capture" in str(err.value)
        # these need no buffer: a lookup, and a row that a wave holds
        ctx.code_embed("bf16", e.table, 500, e.dim, e.dim, 1, 4, e.codes, e.positions, 1, 2.0, "bf16", e.rows, e.dim)
        ctx.code_distill("f16", e.scores, e.n, e.k, 900, 1.0, 6, e.tl, e.tc, 6, True, *e.stats)
    graph = Captured(ctx, refused)
    for _ in range(3):
        graph.launch()
        got = e.results()
        ctx.code_distill("f16", e.scores, e.n, e.k, 900, 1.0, 6, e.tl, e.tc, 6, True, *e.stats)
        ctx.sync()
        for a, b in zip(got, e.results()):
            assert np.array_equal(a, b)
    e.calls()
    ctx.sync()
    graph.close()
    ctx.close()


def test_a_smaller_call_after_a_larger_one():
    """No size of the second call is above the first's: it is captured all the same, whichever way its rows go."""
    import vq_amd
    rng = np.random.default_rng(5)
    for before, then in ((dict(n=64, k=70000, positions=40000), dict(n=63, k=65536, positions=33000)), (dict(n=400, k=40000, positions=33000), dict(n=63, k=39999, positions=32768)),
                         (dict(n=2000, k=16385, positions=2000), dict(n=4, k=16385, positions=1025))):
        ctx = vq_amd.Context(0)
        a, b = Everything(ctx, rng, **before), Everything(ctx, rng, **then)
        a.calls()
        ctx.sync()
        graph = Captured(ctx, b.calls)
        for _ in range(2):
            graph.launch()
            got = b.results()
            a.calls()
            b.calls()
            ctx.sync()
            for x, y in zip(got, b.results()):
                assert np.array_equal(x, y)
        graph.close()
        ctx.close()


def test_fewer_rows_go_another_way():
    """64 rows of 40,000 codes lie in registers, 63 go in parts; 512 sequences of many drafts go at once, 3 in three launches: the smaller calls are
    captured after the larger ones alone."""
    import vq_amd
    rng = np.random.default_rng(11)
    n, k, top = 64, 40000, 4
    ctx = vq_amd.Context(0)
    scores, grad, g = ctx.to_device(rng.standard_normal((n, k)).astype(np.float32)), ctx.empty((n, k), np.float32), ctx.to_device(rng.random(n).astype(np.float32))
    lp, code = ctx.to_device(np.full((n, top), -1.5, np.float32)), ctx.to_device(rng.integers(0, k, (n, top)).astype(np.int32))
    loss = ctx.empty(n, np.float32)

    def call(rows):
        ctx.code_distill("f32", scores, rows, k, k, 1.0, top, lp, code, top, True, loss, None, None, None, g, grad, k)
    call(n)
    ctx.sync()
    graph = Captured(ctx, lambda: call(n - 1))
    for _ in range(3):
        graph.launch()
        a = [loss.download()[:n - 1], grad.download()[:n - 1]]
        call(n)
        call(n - 1)
        assert np.array_equal(a[0], loss.download()[:n - 1]) and np.array_equal(a[1], grad.download()[:n - 1])
    graph.close()
    ctx.close()
    ctx = vq_amd.Context(0)
    n, draft, k = 512, 20, 100
    target, u = ctx.to_device(rng.standard_normal((n * (draft + 1), k)).astype(np.float32)), ctx.to_device(rng.random((n, draft + 1)).astype(np.float32))
    codes, accepted, out = ctx.to_device(rng.integers(0, k, (n, draft)).astype(np.int32)), ctx.empty(n, np.int32), ctx.empty((n, draft + 1), np.int32)

    def verify(count):
        ctx.code_verify("f32", target, k, 1.0, None, k, 1.0, count, draft, k, 4, codes, draft, u, draft + 1, accepted, out, draft + 1)
    verify(n)
    ctx.sync()
    want = out.download()
    graph = Captured(ctx, lambda: verify(3))
    for _ in range(3):
        out.upload(np.zeros((n, draft + 1), np.int32))
        graph.launch()
        assert np.array_equal(out.download()[:3], want[:3]) and not out.download()[3:].any()
        verify(n)
    graph.close()
    ctx.close()


def test_two_contexts_side_by_side():
    """Calls of two contexts in turn, without waiting for one another: each has its own buffers and stream."""
    import vq_amd
    a, b = vq_amd.Context(0), vq_amd.Context(0)
    ea, eb = Everything(a, np.random.default_rng(6)), Everything(b, np.random.default_rng(7), n=33, k=17000)
    ea.calls(), a.sync()
    eb.calls(), b.sync()
    wa, wb = ea.results(), eb.results()
    for _ in range(3):
        for _ in range(5):
            ea.calls()
            eb.calls()
        a.sync(), b.sync()
        for x, y in zip(wa + wb, ea.results() + eb.results()):
            assert np.array_equal(x, y)
    a.close()
    b.close()


def test_refusals_leave_the_context_usable(ctx):
    import vq_amd
    x, c, f = ctx.to_device(np.zeros((4, 8), np.float32)), ctx.to_device(np.zeros(8, np.int32)), ctx.empty(64, np.float32)
    i = ctx.empty(64, np.int32)
    for call in (lambda: ctx.code_embed("f32", x, 4, 8, 9, 1, 4, c, 2, 1, 1.0, "f32", f, 8), lambda: ctx.code_embed("f32", x, 4, 8, 8, 1, 3, c, 2, 1, 1.0, "f32", f, 8),
                 lambda: ctx.code_embed_grad("f32", x, 4, 8, 8, 1, 4, c, 1, float("nan"), 4, False, "f32", f, 8),
                 lambda: ctx.code_distill("f32", x, 4, 8, 8, 0.0, 1, f, c, 1, False, f, None, None, None), lambda: ctx.code_distill("f32", x, 4, 8, 8, 1.0, 65, f, c, 65, False, f, None, None, None),
                 lambda: ctx.code_distill_grad("f32", x, 4, 8, 8, 1.0, 1, f, c, 1, True, f, f, None, f, x, 8),
                 lambda: ctx.code_verify("f32", x, 8, 1.0, None, 8, 1.0, 4, 64, 8, 4, c, 64, f, 65, i, i, 65)):
        with pytest.raises(vq_amd.VqError) as e:
            call()
        assert "Invalid parameter" in str(e.value)
    ctx.code_embed("f32", x, 4, 8, 8, 1, 4, c, 2, 1, 1.0, "f32", f, 8)
    assert not f.download()[:16].any()
