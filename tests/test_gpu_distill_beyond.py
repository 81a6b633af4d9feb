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


def masked_rows(rng, n, k, kind, far):
    """Rows whose codes all have the score `far`, but for two of them, the teacher's alternatives, with 0.5 and 0.3."""
    x = np.full((n, k), far)
    code = np.stack([rng.permutation(k)[:2] for _ in range(n)]).astype(np.int32)
    x[np.arange(n)[:, None], code] = R.unpack(R.pack(rng.uniform(-2, 2, (n, 2)), kind), kind)
    lp = np.log(np.tile(np.array([[0.5, 0.3]]), (n, 1))).astype(np.float32)
    return x, lp, code


def formulas(x, beta, lp, code, g):
    """(loss, log R, gradient) of rows with a rest that has far less than the alternatives: R is nothing beside them, shares of it are not."""
    n, k = x.shape
    rows = np.arange(n)[:, None]
    named = np.zeros((n, k), bool)
    named[rows, code] = True
    q = np.exp(lp.astype(np.float64))
    r = 1.0 - q.sum(axis=1)
    z = beta * x[rows, code]
    top = z.max(axis=1, keepdims=True)
    logp = z - top - np.log(np.exp(z - top).sum(axis=1, keepdims=True))
    L = np.log(np.exp(z - top).sum(axis=1))
    other = np.where(named, -np.inf, beta * (x - x[rows, code].max(axis=1, keepdims=True)))
    most = other.max(axis=1, keepdims=True)
    e = np.exp(other - most)
    logr = most[:, 0] + np.log(e.sum(axis=1)) - L
    loss = (q * (lp - logp)).sum(axis=1) + r * (np.log(r) - logr)
    y = -r[:, None] * e / e.sum(axis=1, keepdims=True)
    y[rows, code] = np.exp(logp) - q
    return loss, logr, y * (beta * g.astype(np.float64))[:, None]


FAR = [("f32", 2.0, LOW["f32"]), ("f32", 1e6, LOW["f32"]), ("bf16", 1.5, LOW["bf16"]), ("bf16", 2.5, LOW["bf16"]), ("f32", 1e30, -1e9)]


@pytest.mark.parametrize("kind,beta,far", FAR)
@pytest.mark.parametrize("k,n", WAYS)
def test_a_rest_below_binary32(ctx, k, n, kind, beta, far):
    """All codes but the alternatives masked by the type's lowest value: log R is beyond binary32, and still they can be, so that the loss has the rest's
    term and the gradient its class."""
    rng = np.random.default_rng(k)
    x, lp, code = masked_rows(rng, n, k, kind, far)
    if beta == 1e30:  # (differences that beta leaves in the range)
        x[np.arange(n), code[:, 0]], x[np.arange(n), code[:, 1]] = 0.0, -1e-30
    beta = float(np.float32(beta))
    g = (rng.random(n) / beta).astype(np.float32)
    if beta == float(np.float32(1e6)):
        x[np.arange(n)[:, None], code] /= 1e6
        x = R.unpack(R.pack(x, kind), kind)
    loss, m, L, lr, y = run(ctx, x, kind, beta, lp, code, True, g, False)
    want, logr, wy = formulas(x, beta, lp, code, g)
    assert (logr < LOW["f32"]).all() and (lr == LOW["f32"]).all()
    # the rest's term is nearly all of the loss: r from two exponentials in f64, rounded once; the product and the sum, once each
    fits = want < 3.4e38
    assert np.isinf(loss[~fits]).all() and (loss[~fits] > 0).all()
    assert (np.abs(loss - want)[fits] <= 8 * U * want[fits]).all()
    rows = np.arange(n)[:, None]
    # p: an exponent of at most 4 rounded four times, two steps of the power, four sums and products; q: rounded once
    tol = beta * g.astype(np.float64)[:, None] * (64 * U)
    near = np.abs(y - wy)[rows, code]
    assert (near <= tol + 1.01 * R.HALF_STEP[kind] * np.abs(wy[rows, code]) + 2.0 ** -126).all()


@pytest.mark.parametrize("rest", [False, True])
@pytest.mark.parametrize("k,n", WAYS)
def test_an_alternative_below_binary32(ctx, k, n, rest):
    """An alternative whose score is masked by the lowest value: its log probability is beyond binary32, its share of the loss is not."""
    rng = np.random.default_rng(k)
    x = R.unpack(R.pack(rng.standard_normal((n, k)), "f32"), "f32")
    code = np.stack([rng.permutation(k)[:2] for _ in range(n)]).astype(np.int32)
    x[np.arange(n), code[:, 1]] = LOW["f32"]
    lp = np.log(np.tile(np.array([[0.9, 0.1]]), (n, 1))).astype(np.float32)
    loss, *_ = run(ctx, x, "f32", 4.0, lp, code, rest, np.ones(n, np.float32), False)
    # q of 0.1: the exponential rounded once, over a sum (a reciprocal, a product), and its product
    want = np.exp(lp[:, 1].astype(np.float64)) / (1.0 if rest else np.exp(lp.astype(np.float64)).sum(axis=1)) * 4.0 * -LOW["f32"]
    assert (np.abs(loss - want) <= 8 * U * want).all()


@pytest.mark.parametrize("kind,beta,far", FAR + [("f32", 1.0, -1e8), ("f32", 1.0, -1e5), ("bf16", 1.0, -1e6), ("f16", 1.0, -60000.0), ("f32", 0.5, -300.0)])
@pytest.mark.parametrize("k,n", WAYS)
def test_shares_of_a_far_rest(ctx, k, n, kind, beta, far):
    """The rest's codes share its gradient, however little they have, where the gradient comes with the loss, in whatever way a row goes; in a call of
    its own to log R's accuracy, and below -2^20 not at all."""
    rng = np.random.default_rng(k + 1)
    x, lp, code = masked_rows(rng, n, k, kind, far)
    rows = np.arange(n)[:, None]
    if beta > 100:
        x[rows, code] /= beta
    else:  # codes among the masked ones that have more of the rest than the others
        odd = rng.random((n, k)) < 0.3
        odd[rows, code] = False
        x[odd] = R.unpack(R.pack(np.array([far * 0.999999]), kind), kind) if far > -1e30 else far
    x = R.unpack(R.pack(x, kind), kind)
    beta = float(np.float32(beta))
    g = (rng.random(n) / beta).astype(np.float32)
    _, logr, wy = formulas(x, beta, lp, code, g)
    named = np.zeros((n, k), bool)
    named[rows, code] = True
    bg = beta * g.astype(np.float64)[:, None]
    # an exponent relative to the rest's largest score, of a difference and a factor rounded once each, and the logarithm of a sum of k terms (each a power
    # of two roundings' exponent), itself to a step of at most 20; the factor r from f64
    d = np.where(named, 0.0, beta * np.abs(x - np.where(named, -np.inf, x).max(axis=1, keepdims=True)))
    rel = (6 * d.max(axis=1, keepdims=True) + 3 * np.log2(k) + 64 + 16) * U
    for own_call in (False, True):
        y = run(ctx, x, kind, beta, lp, code, True, g, own_call)[4]
        if own_call and (logr < -2.0 ** 20).all():
            assert (y[~named] == 0).all()
            continue
        more = rel + (8 * U * np.abs(logr)[:, None] if own_call else 0.0)
        want = np.where(named, 0.0, wy)
        tol = more * np.abs(want) + 1.01 * R.HALF_STEP[kind] * np.abs(want) * (1 + more) + R.LEAST[kind] + bg * 2.0 ** -126
        assert (np.abs(np.where(named, 0.0, y) - want) <= tol).all(), (np.abs(np.where(named, 0.0, y) - want) / np.where(want == 0, 1, np.abs(want))).max()
        if not own_call or (logr > -2.0 ** 20).all():
            # the rest's codes have minus r in all
            total = np.where(named, 0.0, y).sum(axis=1)
            assert (np.abs(total - want.sum(axis=1)) <= tol.sum(axis=1)).all()
