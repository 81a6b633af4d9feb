"""GPU: rows of scores against a teacher where numbers leave binary32: log probabilities above zero, log probabilities and log R below its lowest
number.  Through the C ABI, against the formulas in 64 bits."""
import numpy as np
import pytest

import codes_ref as Q
import scores_ref as R

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
LOW = {"f32": float(np.finfo(np.float32).min), "bf16": -float(2 ** 127 * (2 - 2 ** -7))}
# rows of a wave, of four, of sixteen (64 rows or more), in parts
WAYS = [(6, 5), (300, 7), (3000, 5), (6000, 5), (20000, 70), (20000, 9), (70001, 9)]


@pytest.fixture(scope="module")
def ctx():
    import vq_amd
    c = vq_amd.Context(0)
    yield c
    c.close()


def run(ctx, x, kind, beta, lp, code, rest, g, own_call):
    """(loss, m, L, log R, gradient): the gradient in the same call or in one of its own."""
    n, k = x.shape
    top = lp.shape[1]
    dx, dl, dc, dg = ctx.to_device(R.pack(x, kind)), ctx.to_device(lp), ctx.to_device(code), ctx.to_device(g)
    out = [ctx.empty(n, np.float32) for _ in range(4)]
    grad = ctx.to_device(R.pack(np.full((n, k), 7.0), kind))
    args = (kind, dx, n, k, k, beta, top, dl, dc, top, rest)
    if own_call:
        ctx.code_distill(*args, *out)
        ctx.code_distill_grad(*args, *out[1:], dg, grad, k)
    else:
        ctx.code_distill(*args, *out, dg, grad, k)
    return [o.download().astype(np.float64) for o in out] + [R.unpack(grad.download(), kind)]


@pytest.mark.parametrize("own_call", [False, True])
@pytest.mark.parametrize("k,n", WAYS)
def test_log_probabilities_above_zero(ctx, k, n, own_call):
    """What no probability has: taken as it is, and beyond binary32 neither the loss nor the entry's gradient is a number that looks ordinary."""
    rng = np.random.default_rng(k)
    x = R.unpack(R.pack(rng.standard_normal((n, k)), "f32"), "f32")
    code = np.stack([rng.permutation(k)[:2] for _ in range(n)]).astype(np.int32)
    g = np.ones(n, np.float32)
    for far in (89.0, 100.0, 708.0, 710.0, 720.0, 750.0, 800.0, 1100.0, 1e4, 1e9, 1e30, 3e38):
        lp = np.full((n, 2), np.log(0.25), np.float32)
        lp[::2, 1] = far
        loss, m, L, lr, y = run(ctx, x, "f32", 1.0, lp, code, True, g, own_call)
        assert not np.isfinite(loss[::2]).any() and not (loss[::2] < 0).any()
        assert not np.isfinite(y[np.arange(0, n, 2), code[::2, 1]]).any()
        want = Q.distill(x[1::2], 1.0, lp[1::2], code[1::2], True)
        assert (np.abs(loss[1::2] - want["loss"]) <= want["tloss"]).all() and np.isfinite(y[1::2]).all()
    lp = np.full((n, 2), 80.0, np.float32)  # still within it
    loss, *_ = run(ctx, x, "f32", 1.0, lp, code, True, g, own_call)
    want = Q.distill(x, 1.0, lp, code, True)
    assert (np.abs(loss - want["loss"]) <= want["tloss"]).all()
