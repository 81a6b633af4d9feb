"""GPU: rows of scores against a teacher's alternatives, loss and gradient, through the C ABI, against plain forms in 64 bits
(codes_ref.py)."""
import numpy as np
import pytest

import codes_ref as Q
import scores_ref as R
from test_gpu_embed import held, near, output, rows_of

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    import vq_amd
    c = vq_amd.Context(0)
    yield c
    c.close()


def case(rng, n, k, top, kind, beta=1.0, spread=2.0):
    """Scores, and a teacher that sees something like them; short lists among the teacher's."""
    x = R.unpack(R.pack(rng.standard_normal((n, k)) * spread, kind), kind)
    z = beta * (x + rng.standard_normal((n, k)))
    lp, code = np.full((n, top), -np.inf, np.float32), np.full((n, top), -1, np.int32)
    t = min(top, k)
    best = np.argsort(-z, axis=1, kind="stable")[:, :t]
    full = z - np.log(np.exp(z - z.max(axis=1, keepdims=True)).sum(axis=1, keepdims=True)) - z.max(axis=1, keepdims=True)
    lp[:, :t], code[:, :t] = np.take_along_axis(full, best, 1), best
    short = np.arange(n) % 5 == 3
    lp[short, (top + 1) // 2:], code[short, (top + 1) // 2:] = -np.inf, -1
    return x, lp, code


def run(ctx, x, kind, beta, lp, code, rest, g=None, how="apart", pad=0, offset=0, outputs=(1, 1, 1, 1), teacher_pad=0):
    """One call, checked.  how: the loss alone ("loss"), the gradient in the same call ("same", "inplace"), or in one of its own after it
    ("apart", "apart_inplace")."""
    n, k = x.shape
    top, ld = lp.shape[1], k + pad
    packed = R.pack(x, kind)
    x = R.unpack(packed, kind)
    ds, ps = held(ctx, packed, ld, offset)
    before_scores = ds.download()
    dlp, plp = held(ctx, lp, top + teacher_pad)
    dcode, pcode = ctx.to_device(np.pad(code, ((0, 1), (0, teacher_pad)), constant_values=5)), None
    out = [ctx.to_device(np.full(n + 1, 7, np.float32)) if o else None for o in outputs]
    args = (kind, ps, n, ld, k, beta, top, plp, dcode, top + teacher_pad, rest)
    inplace = how.endswith("inplace")
    fused = how in ("same", "inplace")
    if how != "loss":
        dg = ctx.to_device(g.astype(np.float32))
        if inplace:
            dy, py, before, ldy, off = ds, ps, before_scores, ld, offset
        else:
            ldy, off = k + offset, pad
            dy, py, before = output(ctx, (n, k), kind, ldy, off)
    if fused:
        ctx.code_distill(*args, *out, dg, py, ldy)
    else:
        ctx.code_distill(*args, *out)
        if how != "loss":
            ctx.code_distill_grad(*args, out[1], out[2], out[3], dg, py, ldy)
    got = [None if o is None else o.download() for o in out]
    for o in got:
        assert o is None or o[n] == 7
    loss, m, L, lr = [None if o is None else o[:n] for o in got]
    want = Q.distill(x, beta, lp, code, rest)
    fine = ~want["none"] & ~want["bad"]
    if loss is not None:
        near(loss.astype(np.float64), want["loss"], want["tloss"])
    if m is not None:
        assert np.array_equal(m, want["m"].astype(np.float32), equal_nan=True)
    if L is not None:
        assert np.isnan(L[want["bad"]]).all() and (L[want["none"]] == -np.inf).all() and (L[fine] >= 0).all()
        assert (np.abs(L - want["L"])[fine] <= want["tL"][fine]).all()
    if lr is not None:
        near(lr.astype(np.float64), want["logrest"], want["tlogrest"])
        assert not (lr > 0).any()
    if how == "loss":
        return got
    rows = rows_of(dy, before, (n, k), ldy, off, kind)
    y = R.unpack(rows, kind)
    stats = [a if a is not None else want[name].astype(np.float32) for a, name in zip((m, L, lr), ("m", "L", "logrest"))]
    wy, err = Q.distill_grad(x, beta, lp, code, rest, *stats, g.astype(np.float32))
    near(y, wy, Q.rounded(wy, err, kind))
    if not inplace:
        assert np.array_equal(ds.download().view(np.uint8), before_scores.view(np.uint8))
    return got + [rows]


# rows shorter than a vector of 16 bytes, of a wave with 8 to 64 codes per lane, of four and of sixteen waves, in parts; with odd remainders
LENGTHS = [1, 2, 3, 5, 7, 8, 9, 33, 256, 511, 513, 1001, 1025, 2047, 2500, 4096, 4097, 8190, 8200, 16384, 16385, 20001, 40003]


@pytest.mark.parametrize("kind", R.TYPES)
@pytest.mark.parametrize("k", LENGTHS)
@pytest.mark.parametrize("rest", [False, True])
def test_loss_and_gradient(ctx, k, kind, rest):
    rng = np.random.default_rng(k)
    n = 9 if k > 5000 else 37
    for top, how, beta in ((1, "apart", 1.0), (5, "same", 0.5), (64, "inplace", 1.5), (20, "apart_inplace", 1.0), (3, "loss", 2.0)):
        x, lp, code = case(rng, n, k, top, kind, beta)
        run(ctx, x, kind, beta, lp, code, rest, rng.standard_normal(n), how, pad=k % 5, offset=top % 3, teacher_pad=top % 2)


@pytest.mark.parametrize("kind", R.TYPES)
@pytest.mark.parametrize("k", [16385, 30000, 32768, 32769, 50021, 65536, 65537, 100003])
def test_rows_of_sixteen_waves_and_beyond(ctx, k, kind):
    """64 rows or more, so that the gradient comes from the registers that held the row up to 65,536 codes."""
    rng = np.random.default_rng(k)
    x, lp, code = case(rng, 64, k, 20, kind)
    g = rng.standard_normal(64)
    a = run(ctx, x, kind, 1.0, lp, code, True, g, "same", pad=3)
    run(ctx, x, kind, 1.0, lp, code, True, g, "inplace")
    run(ctx, x, kind, 1.0, lp, code, False, g, "apart", outputs=(1, 1, 1, 0))
    run(ctx, x, kind, 1.0, lp, code, False, g, "same", outputs=(0, 0, 0, 0))
    assert a[0] is not None


WAYS = [6, 300, 900, 3000, 6000, 20000, 50001]


def edge_rows(rng, n, k, kind):
    """Rows of everything: masked codes, -inf only, the type's lowest value as a mask, NaN, +inf, one code far above."""
    x = R.unpack(R.pack(rng.standard_normal((n, k)) * 3, kind), kind)
    low = {"f32": np.finfo(np.float32).min, "f16": -65504.0, "bf16": -float(2 ** 127 * (2 - 2 ** -7))}[kind]
    x[0, rng.random(k) < 0.5] = -np.inf
    x[1] = -np.inf
    x[2, rng.random(k) < 0.7] = low
    x[3, :] = low
    x[4, k // 2] = np.nan
    x[5, k - 1] = np.inf
    x[6, 0] = 60000.0
    x[7, :] = -np.inf
    x[7, k // 3] = 1.0
    x[8, :] = 0.25
    x[9, :] = -np.inf
    x[9, 0] = low
    return x


@pytest.mark.parametrize("kind", R.TYPES)
@pytest.mark.parametrize("k", WAYS)
@pytest.mark.parametrize("rest", [False, True])
def test_rows_at_the_edges(ctx, k, kind, rest):
    rng = np.random.default_rng(k)
    n = 70 if k == 20000 else 14
    top = 4
    x = edge_rows(rng, n, k, kind)
    for spread in (False, True):
        lp = np.log(np.array([0.4, 0.3, 0.15, 0.05], np.float32))[None].repeat(n, 0).astype(np.float32)
        code = np.stack([rng.permutation(k)[:top] if k >= top else np.arange(top) for _ in range(n)]).astype(np.int32)
        if spread:
            code[:, 0] = np.where(np.arange(n) < 10, [0, 1, 2, 3, k // 2, k - 1, 0, k // 3, 4, 0][0:10] + [0] * (n - 10), code[:, 0]) % k
            code[10, 1] = code[10, 0]  # the same code twice
            code[11, :] = -1           # no teacher
            lp[12, 0], code[12, 0] = -np.inf, k + 7  # an entry without probability is none, whatever its code
        for how in ("same", "apart", "inplace"):
            if kind == "f32" and how == "apart":
                x[13, 1] = -1e38
            run(ctx, x, kind, 1.0, lp, code, rest, rng.standard_normal(n), how)
            run(ctx, x, kind, 0.25, lp, code, rest, rng.standard_normal(n), how, pad=1)


@pytest.mark.parametrize("kind", R.TYPES)
@pytest.mark.parametrize("k", WAYS)
@pytest.mark.parametrize("rest", [False, True])
def test_teachers_at_the_edges(ctx, k, kind, rest):
    """Lists with codes out of range, NaN and +inf, no entries, one code throughout, certainty, probabilities too small to count, more than one in all."""
    rng = np.random.default_rng(k)
    n, top = 12, 5
    x = R.unpack(R.pack(rng.standard_normal((n, k)), kind), kind)
    lp = np.full((n, top), np.log(0.15), np.float32)
    code = np.tile(np.arange(top, dtype=np.int32) % k, (n, 1))
    code[0, 2] = k
    code[1, 4] = 2 ** 31 - 1
    lp[2, 1] = np.nan
    lp[3, 3] = np.inf
    code[4] = -1
    lp[5] = -np.inf
    code[6] = k - 1
    lp[7], code[7, 1:] = 0.0, -1           # certain
    lp[8] = -np.array([0.1, 50, 120, 500, 5000])
    lp[9] = np.log(0.5)                    # two and a half in all
    lp[10, 0], code[10, 0] = np.nan, -1    # a negative code is none, whatever its log probability
    x[4, 0] = np.nan                       # no teacher: zero, whatever the scores
    for how in ("same", "apart", "inplace", "loss"):
        run(ctx, x, kind, 1.0, lp, code, rest, rng.standard_normal(n), how)


@pytest.mark.parametrize("kind", R.TYPES)
@pytest.mark.parametrize("k", [4, 12, 64])
def test_every_code_an_alternative(ctx, k, kind):
    """Nothing is left: no class beside the alternatives."""
    rng = np.random.default_rng(k)
    x, lp, code = case(rng, 20, k, k, kind)
    for how in ("same", "apart"):
        got = run(ctx, x, kind, 1.0, lp, code, True, rng.standard_normal(20), how)
        full = np.arange(20) % 5 != 3
        assert (got[3][:20][full] == -np.inf).all() and np.isfinite(got[0][:20]).all()


def test_far_scores_and_betas(ctx):
    """Scores and betas whose products are far from 1, in every way a row goes."""
    rng = np.random.default_rng(4)
    for k in WAYS:
        for spread, beta in ((1e4, 1e-4), (1e-4, 1e4), (3e37, 1e-30), (1e3, 1.0)):
            x, lp, code = case(rng, 6, k, min(5, k), "f32", beta, spread)
            x += 20 * spread
            x = x.astype(np.float32).astype(np.float64)
            beta = float(np.float32(beta))
            run(ctx, x, "f32", beta, lp, code, True, np.full(6, 1 / beta), "same")


def test_a_student_like_its_teacher_has_no_loss(ctx):
    """The teacher's own scores against its alternatives: the loss is zero, and the gradient, up to their rounding."""
    rng = np.random.default_rng(6)
    n, k, top = 50, 3000, 20
    x = rng.standard_normal((n, k)).astype(np.float32)
    dx, lp, code = ctx.to_device(x), ctx.empty((n, top), np.float32), ctx.empty((n, top), np.int32)
    ctx.code_logprobs("f32", dx, n, k, k, 1.0, 4, None, 1, top, None, None, None, None, lp, code)
    loss, grad, g = ctx.empty(n, np.float32), ctx.empty((n, k), np.float32), ctx.to_device(np.ones(n, np.float32))
    ctx.code_distill("f32", dx, n, k, k, 1.0, top, lp, code, top, True, loss, None, None, None, g, grad, k)
    # log probabilities and sums are rounded a few times each; 20 below zero at most
    assert np.abs(loss.download()).max() < 40 * 20 * Q.U24 and np.abs(grad.download()).max() < 40 * 20 * Q.U24


@pytest.mark.parametrize("k", [50, 3000, 20000])
def test_gradient_against_differences(ctx, k):
    """The kernels' gradient against the plain loss's central differences, in 64 bits."""
    rng = np.random.default_rng(k)
    n, h = 3, 1e-4
    for rest in (False, True):
        x, lp, code = case(rng, n, k, 5, "f32")
        y = R.unpack(run(ctx, x, "f32", 1.0, lp, code, rest, np.ones(n), "same")[4], "f32")
        for j in [0, k - 1, *code[0, :3], *rng.integers(0, k, 5)]:
            if j < 0:
                continue
            e = np.zeros(k)
            e[j] = h
            d = (Q.distill(x + e, 1.0, lp, code, rest)["loss"] - Q.distill(x - e, 1.0, lp, code, rest)["loss"]) / (2 * h)
            # the difference is off by h^2 / 6 of the third derivative, which is below 1, and by 1e-16 / h of the loss
            assert np.abs(d - y[:, j]).max() < 2e-9 + 1e-11 + 1e-6 * np.abs(d).max()


@pytest.mark.parametrize("kind", R.TYPES)
def test_most_codes(ctx, kind):
    rng = np.random.default_rng(30)
    x, lp, code = case(rng, 2, 1 << 20, 64, kind)
    for rest, how in ((True, "same"), (False, "inplace")):
        run(ctx, x, kind, 1.0, lp, code, rest, rng.standard_normal(2), how)


def test_more_rows_than_a_launch_takes(ctx):
    """Short rows, of which a launch takes 2^25."""
    n, k = (1 << 25) + 5, 2
    x = np.zeros((n, k), np.float32)
    x[:, 1] = np.arange(n) % 7
    lp, code = np.full((n, 1), -0.5, np.float32), np.ones((n, 1), np.int32)
    loss = ctx.empty(n, np.float32)
    ctx.code_distill("f32", ctx.to_device(x), n, k, k, 1.0, 1, ctx.to_device(lp), ctx.to_device(code), 1, False, loss, None, None, None)
    want = Q.distill(x[:7].astype(np.float64), 1.0, lp[:7], code[:7], False)
    got = loss.download()
    for i in range(7):
        assert (np.abs(got[i::7] - want["loss"][i]) <= want["tloss"][i]).all()


@pytest.mark.parametrize("kind", R.TYPES)
@pytest.mark.parametrize("k", [300, 900, 3000, 6000, 20001, 65537])
def test_alternatives_that_hold_next_to_nothing(ctx, k, kind):
    """log R, next to zero, and what the other codes' gradients have in common, a difference of two small shares, to the number's own
    accuracy: both come of the alternatives' own sum."""
    rng = np.random.default_rng(k)
    n, top, u = 70, 3, 2.0 ** -24
    x = R.unpack(R.pack(rng.standard_normal((n, k)), kind), kind)
    code = np.stack([rng.permutation(k)[:top] for _ in range(n)]).astype(np.int32)
    rows = np.arange(n)[:, None]
    x[rows, code] = R.unpack(R.pack(rng.uniform(-4, -2, (n, top)), kind), kind)
    d = x - x.max(axis=1, keepdims=True)
    e = np.exp(d)
    S = e.sum(axis=1)
    share = e[rows, code].sum(axis=1) / S
    lp = np.log(e[rows, code] / S[:, None] * rng.uniform(2, 3, (n, top))).astype(np.float32)
    g = (rng.random(n) + 0.5).astype(np.float32)
    for how in ("same", "apart"):
        got = run(ctx, x, kind, 1.0, lp, code, True, g, how)
        lr, y = got[3][:n].astype(np.float64), R.unpack(got[4], kind)
        want = np.log1p(-share)
        # a term: the product's, the factor's and the difference's rounding times its exponent, and the power's; two sums, of three and (tL) of k
        # terms, a reciprocal, a product; log1p makes at most 1.5 times as much of that and adds two steps
        tL = Q.distill(x, 1.0, lp, code, True)["tL"]
        rel = 1.5 * ((3 * np.abs(d[rows, code]).max(axis=1) + 12) * u + tL) + 4 * u
        assert (np.abs(lr - want) <= rel * np.abs(want)).all()
        q = np.exp(lp.astype(np.float64)).sum(axis=1)
        factor = q - share  # Q R - r, where Q + r are one
        wy = g.astype(np.float64)[:, None] * factor[:, None] * e / (S * (1 - share))[:, None]
        # the factor: of a log R that is off by rel, a power less one, a product, a rounded Q, a sum; the share: as in distill_grad
        L = np.log(S)[:, None]
        ep = (6 * np.abs(d) + 4 * np.abs(d - L) + 8 * L + 24) * u + 2 * tL[:, None]
        err = 1.01 * np.abs(wy) * (((rel + 8 * u) * share + 8 * u * q)[:, None] / np.abs(factor)[:, None] + ep) + 2.0 ** -126
        other = np.ones((n, k), bool)
        other[rows, code] = False
        near(np.where(other, y, 0.0), np.where(other, wy, 0.0), Q.rounded(wy, err, kind))


def test_a_loss_of_next_to_nothing(ctx):
    """Alternatives of a few billionths, and the teacher's of as little: r log r and r log R are small, and so is what they leave."""
    k, n = 4096, 8
    x = np.zeros((n, k))
    x[:, 5] = -np.arange(8, 16)
    code = np.full((n, 1), 5, np.int32)
    share = np.exp(x[:, 5]) / (k - 1 + np.exp(x[:, 5]))
    lp = np.log(3 * share).astype(np.float32)[:, None]
    got = run(ctx, x, "f32", 1.0, lp, code, True, how="loss")
    q = np.exp(lp[:, 0].astype(np.float64))
    parts = q * (lp[:, 0] - np.log(share)), (1 - q) * (np.log1p(-q) - np.log1p(-share))
    # log p_c: a product and a difference (exact here), L's rounding, theirs; the rest's two logarithms are relative to their own size: log R's
    # share has the exponent's two roundings (15 at most), a power's, a sum's, a reciprocal's and a product's
    err = q * 2.0 ** -24 * (4 * np.abs(np.log(share)) + 32) + 2.0 ** -24 * (48 * share + 8 * q)
    assert (np.abs(got[0][:n] - sum(parts)) <= err).all()
