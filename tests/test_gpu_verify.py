"""GPU: drafted codes against a model's probabilities and the code that comes next, through the C ABI, against plain forms in 64 bits
(codes_ref.py).  Outcomes are whole numbers and have to be equal."""
import numpy as np
import pytest

import codes_ref as Q
import scores_ref as R
from test_gpu_embed import device_codes, held, output

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    import vq_amd
    c = vq_amd.Context(0)
    yield c
    c.close()


def case(rng, n, draft, k, kind, beta, beta_draft, scored=True, spread=2.0, noise=0.7, masked=0.0):
    t = rng.standard_normal((n, draft + 1, k)) * spread
    if masked:
        gone = rng.random((n, draft + 1, k)) < masked
        gone[:, :, 0] = False
        t[gone] = -np.inf
    t = R.unpack(R.pack(t, kind), kind)
    d = R.unpack(R.pack(t[:, :draft] + rng.standard_normal((n, draft, k)) * noise, kind), kind)
    z = beta_draft * d
    codes = (z + rng.gumbel(size=z.shape)).argmax(axis=2) if draft else np.zeros((n, 0), np.int64)
    u = rng.random((n, draft + 1)).astype(np.float32)
    return t, d if scored else None, codes, u


def run(ctx, t, d, codes, u, kind, beta, beta_draft, nbytes=4, pad=0, offset=0):
    n, rows, k = t.shape
    draft = rows - 1
    dt, pt = held(ctx, R.pack(t.reshape(n * rows, k), kind), k + pad, offset)
    dd, pd = (None, None) if d is None else held(ctx, R.pack(d.reshape(n * draft, k), kind), k + pad + 1, offset)
    dc, pc = device_codes(ctx, codes, nbytes, draft + pad, 1) if draft else (None, None)
    du, pu = held(ctx, u, rows + pad)
    da = ctx.to_device(np.full(n + 1, 77, np.int32))
    do = ctx.to_device(np.full((n + 1, rows + pad), 77, np.int32))
    ctx.code_verify(kind, pt, k + pad, beta, pd, k + pad + 1, beta_draft, n, draft, k, nbytes, pc, draft + pad, pu, rows + pad, da, do, rows + pad)
    accepted, out = da.download(), do.download()
    assert accepted[n] == 77 and (out[n] == 77).all() and (out[:, rows:] == 77).all()
    accepted, out = accepted[:n], out[:n, :rows]
    wa, wo = Q.verify(t, float(np.float32(beta)), d, float(np.float32(beta_draft)), codes, u.astype(np.float64))
    assert np.array_equal(accepted, wa), (accepted[accepted != wa][:5], wa[accepted != wa][:5], np.nonzero(accepted != wa)[0][:5])
    assert np.array_equal(out, wo), (out[(out != wo).any(axis=1)][:3], wo[(out != wo).any(axis=1)][:3])
    return accepted, out


LENGTHS = [1, 2, 3, 5, 7, 8, 15, 16, 17, 255, 256, 1001, 4095, 4096, 4097, 8193, 50021]


@pytest.mark.parametrize("kind", R.TYPES)
@pytest.mark.parametrize("scored", [True, False])
@pytest.mark.parametrize("k", LENGTHS)
def test_verify(ctx, k, kind, scored):
    rng = np.random.default_rng(k)
    n = 5 if k > 5000 else 40
    for draft, beta, beta_draft in ((0, 1.0, 1.0), (1, 0.5, 1.0), (4, 1.0, 0.75), (7, 1.5, 1.5)):
        t, d, codes, u = case(rng, n, draft, k, kind, beta, beta_draft, scored)
        run(ctx, t, d, codes, u, kind, beta, beta_draft, 4, pad=draft % 3, offset=draft % 2)


@pytest.mark.parametrize("nbytes", [1, 2, 4])
def test_widths_of_codes(ctx, nbytes):
    rng = np.random.default_rng(nbytes)
    k = 256 if nbytes == 1 else 3000
    for scored in (True, False):
        t, d, codes, u = case(rng, 30, 3, k, "bf16", 1.0, 1.0, scored)
        codes[:, 0] = k - 1
        run(ctx, t, d, codes, u, "bf16", 1.0, 1.0, nbytes)


@pytest.mark.parametrize("scored", [True, False])
def test_drafts_of_different_lengths(ctx, scored):
    rng = np.random.default_rng(5)
    t, d, codes, u = case(rng, 200, 5, 300, "f32", 1.0, 1.0, scored, noise=0.2)
    for b in range(200):
        codes[b, rng.integers(0, 6):] = -1
    codes[7] = [1, -1, 2, 3, 4]  # what is behind the first that is none counts for nothing
    a, out = run(ctx, t, d, codes, u, "f32", 1.0, 1.0)
    assert len(set(a)) > (3 if scored else 1)  # (a draft without scores stays with its code's probability, about 1 in 300)


@pytest.mark.parametrize("kind", R.TYPES)
@pytest.mark.parametrize("scored", [True, False])
def test_masked_codes(ctx, kind, scored):
    rng = np.random.default_rng(11)
    for k in (9, 700, 9000):
        t, d, codes, u = case(rng, 30, 3, k, kind, 1.0, 1.0, scored, masked=0.6)
        codes[3, 0] = np.nonzero(t[3, 0] == -np.inf)[0][0] if (t[3, 0] == -np.inf).any() else codes[3, 0]
        t[4, 1] = -np.inf
        t[4, 1, k // 2] = 3.0  # one code that can be
        run(ctx, t, d, codes, u, kind, 1.0, 1.0)


@pytest.mark.parametrize("kind", R.TYPES)
@pytest.mark.parametrize("scored", [True, False])
@pytest.mark.parametrize("k", [6, 500, 9001])
def test_rows_that_cannot_be_answered(ctx, k, kind, scored):
    rng = np.random.default_rng(k)
    n, draft = 16, 2
    t, d, codes, u = case(rng, n, draft, k, kind, 1.0, 1.0, scored, noise=0.1)
    u[:, :draft] *= 0.3  # most drafts stay
    low = {"f32": np.finfo(np.float32).min, "f16": -65504.0, "bf16": -float(2 ** 127 * (2 - 2 ** -7))}[kind]
    t[0, 0], t[1, 1], t[2, 2] = -np.inf, -np.inf, -np.inf
    t[3, 0, k // 2], t[4, 1, k - 1], t[5, 2, 0] = np.nan, np.inf, np.nan
    t[6, 0], t[7, 1, 1:] = low, low
    codes[8, 0], codes[9, 1] = k, 2 ** 31 - 1
    t[12, 0] = -np.inf
    t[12, 0, codes[12, 0]] = 0.5
    t[13, 0, codes[13, 0]] = np.nan
    t[14, 0, codes[14, 0]] = np.inf
    t[15, 0, codes[15, 0]] = -np.inf
    if scored:
        d[10, 0], d[11, 1, 0] = -np.inf, np.nan
        d[6, 0] = low
    run(ctx, t, d, codes, u, kind, 1.0, 1.0)


def test_random_numbers_at_their_ends(ctx):
    rng = np.random.default_rng(3)
    for k in (7, 5000):
        for scored in (True, False):
            t, d, codes, u = case(rng, 12, 2, k, "f32", 1.0, 1.0, scored, masked=0.3)
            most = np.float32(1.0) - np.float32(2.0 ** -24)
            u[0], u[1], u[2, :2], u[2, 2], u[3, :2], u[3, 2] = 0.0, most, 0.0, most, most, 0.0
            u[4, 2], u[5, 2] = 1.0, 2.0  # beyond the range: the last code that can be
            run(ctx, t, d, codes, u, "f32", 1.0, 1.0)


def test_a_draft_from_the_target_s_own_scores_stays(ctx):
    rng = np.random.default_rng(2)
    t, d, codes, u = case(rng, 50, 4, 700, "f16", 1.0, 1.0, noise=0.0)
    a, out = run(ctx, t, d, codes, u, "f16", 1.0, 1.0)
    assert (a == 4).all() and np.array_equal(out[:, :4], codes) and (out[:, 4] >= 0).all()


def test_longest_drafts(ctx):
    rng = np.random.default_rng(63)
    for scored in (True, False):
        t, d, codes, u = case(rng, 4, 63, 5000, "bf16", 1.0, 1.0, scored, noise=0.05)
        u[0, :63] = 0.0
        run(ctx, t, d, codes, u, "bf16", 1.0, 1.0)


def test_far_scores_and_betas(ctx):
    rng = np.random.default_rng(4)
    for spread, beta in ((1e4, 1e-4), (1e-4, 1e4), (3e37, 1e-30), (1e3, 1.0), (1e30, 1.0)):
        t, d, codes, u = case(rng, 20, 3, 5000, "f32", beta, beta, spread=spread, noise=0.5 * spread)
        run(ctx, t, d, codes, u, "f32", beta, beta)


def test_more_sequences_than_a_launch_takes(ctx):
    """2^23 parts of rows are a launch's: 1.4 million sequences of three rows each take two."""
    rng = np.random.default_rng(1)
    n, k = (1 << 23) // 3 + 1000, 3
    t, d, codes, u = case(rng, 1000, 1, k, "f32", 1.0, 1.0)
    tile = lambda a: np.ascontiguousarray(np.concatenate([a] * (n // 1000 + 1))[:n])
    t2, d2, c2, u2 = tile(t), tile(d), tile(codes).astype(np.int32), tile(u)
    dt, dd, dc, du = ctx.to_device(t2.astype(np.float32)), ctx.to_device(d2.astype(np.float32)), ctx.to_device(c2), ctx.to_device(u2)
    da, do = ctx.empty(n, np.int32), ctx.empty((n, 2), np.int32)
    ctx.code_verify("f32", dt, k, 1.0, dd, k, 1.0, n, 1, k, 4, dc, 1, du, 2, da, do, 2)
    wa, wo = Q.verify(t, 1.0, d, 1.0, codes, u.astype(np.float64))
    assert np.array_equal(da.download(), tile(wa)) and np.array_equal(do.download(), tile(wo))


@pytest.mark.parametrize("kind", R.TYPES)
@pytest.mark.parametrize("scored", [True, False])
@pytest.mark.parametrize("k", [2047, 2048, 2049, 30])
def test_around_the_lines_between_the_ways(ctx, k, kind, scored):
    """Rows of one workgroup per sequence and of parts; many drafts of few and of many sequences."""
    rng = np.random.default_rng(k)
    for n, draft in ((3, 16), (3, 17), (512, 17 if k < 100 else 3)):
        t, d, codes, u = case(rng, n, draft, k, kind, 1.0, 1.0, scored, noise=0.3)
        u[:, :draft] *= 0.5
        run(ctx, t, d, codes, u, kind, 1.0, 1.0, pad=k % 3, offset=1)


def test_enough_rows_for_four_parts_to_a_workgroup(ctx):
    """Masked codes, whole parts among them, where a workgroup makes the sums of four parts of a row."""
    rng = np.random.default_rng(8)
    for kind, k in (("bf16", 17000), ("f32", 40000), ("f16", 5000)):
        n, draft = (2100 if k == 5000 else 700 if k == 17000 else 240), 1
        t, d, codes, u = case(rng, n, draft, k, kind, 1.0, 1.0, spread=1.0)
        t[::3, :, :4096] = -np.inf
        t[1::5, :, 4096:] = -np.inf
        t[5, 0], t[6, 1], t[7, 0, 4500], t[8, 1, 2] = -np.inf, -np.inf, np.nan, np.inf
        u[::4, :draft] = 0.999
        u[9], u[10] = 0.0, 1.0
        run(ctx, t, d, codes, u, kind, 1.0, 1.0)
        run(ctx, t, None, codes, u, kind, 1.0, 1.0)


@pytest.mark.parametrize("scored", [True, False])
def test_most_codes(ctx, scored):
    """More than 64 parts of a row, up to as many as there may be."""
    rng = np.random.default_rng(20)
    for k, n in ((270_001, 3), (1 << 20, 2)):
        t, d, codes, u = case(rng, n, 2, k, "bf16", 1.0, 1.0, scored, noise=0.3)
        t[0, 0, :300_000] = -np.inf
        t[0, 0, k - 1] = 2.0
        run(ctx, t, d, codes, u, "bf16", 1.0, 1.0)
