"""GPU: the operators of models over codes on rows whose places pass 32 bits: a few rows, gigabytes apart in all."""
import numpy as np
import pytest

import codes_ref as Q
import scores_ref as R
from test_gpu_embed import near

pytestmark = pytest.mark.gpu
LD = (1 << 23) + 8


class Far:
    """Rows LD elements apart in memory that is not otherwise looked at."""

    def __init__(self, ctx, n, kind, rows=None):
        import vq_amd
        self.ctx, self.lib, self.item, self.n = ctx, vq_amd._ffi.lib(), 4 if kind == "f32" else 2, n
        self.kind = kind
        self.array = ctx.empty(((n - 1) * LD + 70000,), np.float32 if kind == "f32" else np.uint16 if kind == "bf16" else np.float16)
        self.ptr = self.array.ptr
        if rows is not None:
            for i in range(n):
                row = np.ascontiguousarray(rows[i])
                ctx._check(self.lib.vq_h2d(ctx._h, self.ptr + i * LD * self.item, row.ctypes.data, row.nbytes))

    def rows(self, length):
        out = np.empty((self.n, length), self.array.dtype)
        for i in range(self.n):
            row = np.empty(length, self.array.dtype)
            self.ctx._check(self.lib.vq_d2h(self.ctx._h, row.ctypes.data, self.ptr + i * LD * self.item, row.nbytes))
            out[i] = row
        return out


@pytest.fixture(scope="module")
def ctx():
    import vq_amd
    c = vq_amd.Context(0)
    yield c
    c.close()


@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_tables(ctx, kind):
    """A table, its gradient and the rows of both, each of more than 4 GiB: one stage, and two."""
    rng = np.random.default_rng(1)
    n, dim = 300, 41
    for m, k in ((1, 300), (2, 150)):
        table = R.pack(rng.standard_normal((m * k, dim)), kind)
        codes = rng.integers(0, k, (n, m)).astype(np.int32)
        codes[::17] = -1
        far, out, dc = Far(ctx, m * k, kind, table), Far(ctx, n, kind), ctx.to_device(codes)
        ctx.code_embed(kind, far.ptr, k, LD, dim, m, 4, dc, n, m, 1.5, kind, out.ptr, LD)
        want, err = Q.embed(R.unpack(table, kind).reshape(m, k, dim), codes, 1.5)
        got = out.rows(dim)
        near(R.unpack(got, kind), want, Q.rounded(want, err, kind))
        ctx.code_embed_grad(kind, out.ptr, n, LD, dim, m, 4, dc, m, 0.5, k, False, kind, far.ptr, LD)
        want, err = Q.embed_grad(R.unpack(got, kind), codes, 0.5, k)
        near(R.unpack(far.rows(dim), kind).reshape(m, k, dim), want, Q.rounded(want, err, kind))
        del far, out


@pytest.mark.parametrize("k", [300, 6000, 60000])
def test_rows_of_scores(ctx, k):
    """Rows against a teacher, and drafts, more than 4 GiB apart."""
    rng = np.random.default_rng(k)
    n, top = 140, 5
    x = rng.standard_normal((n, k)).astype(np.float32)
    lp, code = np.log(np.full((n, top), 0.15, np.float32)), np.stack([rng.permutation(k)[:top] for _ in range(n)]).astype(np.int32)
    scores, grad = Far(ctx, n, "f32", x), Far(ctx, n, "f32")
    dl, dc = ctx.to_device(lp), ctx.to_device(code)
    g = rng.random(n).astype(np.float32)
    stats, dg = [ctx.empty(n, np.float32) for _ in range(4)], ctx.to_device(g)
    o = Q.distill(x.astype(np.float64), 1.0, lp, code, True)
    for same in (True, False):
        ctx.code_distill("f32", scores.ptr, n, LD, k, 1.0, top, dl, dc, top, True, *stats, *((dg, grad.ptr, LD) if same else ()))
        if not same:
            ctx.code_distill_grad("f32", scores.ptr, n, LD, k, 1.0, top, dl, dc, top, True, *stats[1:], dg, grad.ptr, LD)
        near(stats[0].download().astype(np.float64), o["loss"], o["tloss"])
        want, err = Q.distill_grad(x.astype(np.float64), 1.0, lp, code, True, *(s.download() for s in stats[1:]), g)
        near(grad.rows(k).astype(np.float64), want, Q.rounded(want, err, "f32"))
    draft = 3
    seq = n // (draft + 1)
    d = Far(ctx, seq * draft, "f32", x[:seq * draft])
    codes = rng.integers(0, k, (seq, draft)).astype(np.int32)
    codes[:, 0] = x[::draft + 1][:seq].argmax(axis=1)
    u = (rng.random((seq, draft + 1)) * 0.3).astype(np.float32)
    accepted, out = ctx.empty(seq, np.int32), ctx.empty((seq, draft + 1), np.int32)
    ctx.code_verify("f32", scores.ptr, LD, 1.0, d.ptr, LD, 0.5, seq, draft, k, 4, ctx.to_device(codes), draft, ctx.to_device(u), draft + 1, accepted, out, draft + 1)
    t = x[:seq * (draft + 1)].reshape(seq, draft + 1, k).astype(np.float64)
    wa, wo = Q.verify(t, 1.0, x[:seq * draft].reshape(seq, draft, k).astype(np.float64), 0.5, codes, u.astype(np.float64))
    assert np.array_equal(accepted.download(), wa) and np.array_equal(out.download(), wo)
