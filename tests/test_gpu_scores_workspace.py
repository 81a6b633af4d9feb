"""GPU: captured calls on log probabilities and 8-bit scores that find the workspace of larger calls before them."""
import ctypes as C

import numpy as np
import pytest

import scores_ref as R

pytestmark = pytest.mark.gpu


class Captured:
    """What `call` issues on a context's stream, as a graph."""

    def __init__(self, ctx, call):
        import vq_amd
        self.hip, self.ctx = C.CDLL("libamdhip64.so"), ctx
        self.stream = C.c_void_p(vq_amd._ffi.lib().vq_ctx_stream(ctx._h))
        self.graph, self.run = C.c_void_p(), C.c_void_p()
        assert self.hip.hipStreamBeginCapture(self.stream, 2) == 0
        try:
            call()
        finally:
            assert self.hip.hipStreamEndCapture(self.stream, C.byref(self.graph)) == 0
        assert self.hip.hipGraphInstantiate(C.byref(self.run), self.graph, None, None, 0) == 0

    def launch(self):
        assert self.hip.hipGraphLaunch(self.run, self.stream) == 0
        self.ctx.sync()

    def close(self):
        assert self.hip.hipGraphExecDestroy(self.run) == 0 and self.hip.hipGraphDestroy(self.graph) == 0


@pytest.mark.parametrize("before,then", [((1024, 65536, 2), (1023, 65536, 2)), ((700, 100_000, 4), (690, 90_000, 3)), ((4097, 16_385, 1), (2047, 16_385, 1)),
                                         ((250, 270_000, 2), (250, 250_000, 2)), ((9, 540_000, 32), (9, 500_000, 31))])
def test_a_smaller_call_after_a_larger_one(before, then):
    """No size of the second call is above the first's, but its rows may go in more parts: it is captured all the same."""
    import vq_amd
    ctx = vq_amd.Context(0)
    n, k, top = before
    x = R.pack(np.random.default_rng(n).standard_normal((61, k)).astype(np.float32), "bf16")
    rows = np.concatenate([x] * (n // 61 + 1))[:n]
    dx, codes = ctx.to_device(rows), ctx.to_device((np.arange(n) % then[1]).astype(np.int32))
    out, tl, tc = [ctx.empty(n, np.float32) for _ in range(4)], ctx.empty((n, top), np.float32), ctx.empty((n, top), np.int32)

    def call(n2, k2, top2):
        ctx.code_logprobs("bf16", dx, n2, k, k2, 1.0, 4, codes, 1, top2, *out, tl, tc)

    def results(n2, k2, top2):
        return [a.download().reshape(-1)[:size].view(np.uint32) for a, size in [(o, n2) for o in out] + [(tl, n2 * top2), (tc, n2 * top2)]]
    call(*before)
    ctx.sync()
    graph = Captured(ctx, lambda: call(*then))
    for _ in range(3):
        graph.launch()
        got = results(*then)
        call(*before)
        call(*then)
        for a, b in zip(got, results(*then)):
            assert np.array_equal(a, b)
    graph.close()
    ctx.close()


def test_fewer_copied_rows_after_more():
    """Rows that are copied to aligned ones: a capture of fewer of them against the same codes."""
    import vq_amd
    ctx = vq_amd.Context(0)
    n, dim, k = 3000, 333, 777
    rng = np.random.default_rng(2)
    x, w = rng.integers(-127, 128, (n, dim)).astype(np.int8), rng.integers(-127, 128, (k, dim)).astype(np.int8)
    xs, ws = rng.uniform(0.001, 0.01, n).astype(np.float32), rng.uniform(0.001, 0.01, k).astype(np.float32)
    dx, dw, dxs, dws, out = ctx.to_device(x), ctx.to_device(w), ctx.to_device(xs), ctx.to_device(ws), ctx.empty((n, k), np.float32)

    def call(rows):
        ctx.scores_i8(dx, dxs, rows, dim, dw, dws, k, dim, dim, None, "f32", out, k)
    call(n)
    ctx.sync()
    few = 1500
    graph = Captured(ctx, lambda: call(few))
    want, tol = R.scores(x[:few], xs[:few], w, ws, None, "f32")
    for _ in range(3):
        out.upload(np.zeros((n, k), np.float32))
        graph.launch()
        got = out.download()
        assert (np.abs(got[:few] - want) <= tol).all() and not got[few:].any()
        call(n)
        ctx.sync()
    graph.close()
    ctx.close()
