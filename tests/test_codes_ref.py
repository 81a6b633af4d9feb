"""The plain 64-bit forms that the kernels of models over codes are held to (codes_ref.py), against differences of what they are the
gradients of, and against frequencies."""
import numpy as np
import pytest

import codes_ref as Q
import scores_ref as R


def _case(rng, n, k, top, dup=False):
    x = rng.standard_normal((n, k)) * 2
    z = x + rng.standard_normal((n, k))
    lp = z - np.log(np.exp(z).sum(axis=1, keepdims=True))
    code = np.argsort(-lp, axis=1)[:, :top]
    if dup:
        code[:, 1] = code[:, 0]
    return x, np.take_along_axis(lp, code, 1).astype(np.float32), code.astype(np.int32)


@pytest.mark.parametrize("rest", [False, True])
@pytest.mark.parametrize("dup", [False, True])
@pytest.mark.parametrize("k,top", [(7, 2), (40, 5), (6, 6)])
def test_gradient_of_the_loss_against_differences(rest, dup, k, top):
    rng = np.random.default_rng(k)
    beta, n = 0.7, 5
    x, lp, code = _case(rng, n, k, top, dup)
    if dup and rest:
        lp = lp - 1.0  # (the entries leave something)
    code[2, 1:] = -1
    lp[3, 0] = -np.inf
    g = rng.standard_normal(n)
    o = Q.distill(x, beta, lp, code, rest)
    y, _ = Q.distill_grad(x, beta, lp, code, rest, o["m"], o["L"], o["logrest"], g)
    h = 1e-5
    for j in range(k):
        e = np.zeros(k)
        e[j] = h
        d = (Q.distill(x + e, beta, lp, code, rest)["loss"] - Q.distill(x - e, beta, lp, code, rest)["loss"]) / (2 * h)
        assert np.abs(d * g - y[:, j]).max() < 1e-8


def test_gradient_of_the_table_is_the_transpose_of_the_lookup():
    rng = np.random.default_rng(3)
    m, k, dim, n = 3, 9, 4, 30
    codes = rng.integers(-1, k, (n, m))
    t, g = rng.standard_normal((m, k, dim)), rng.standard_normal((n, dim))
    y, _ = Q.embed(t, codes, 1.5)
    d, _ = Q.embed_grad(g, codes, 1.5, k)
    assert abs((y * g).sum() - (t * d).sum()) < 1e-10


@pytest.mark.parametrize("scored", [True, False])
def test_verified_codes_have_the_target_s_distribution(scored):
    """Whatever the drafts come from, the first code that is answered has the target's probabilities."""
    rng = np.random.default_rng(5)
    k, n = 6, 40000
    t, d = rng.standard_normal(k), rng.standard_normal(k)
    q = np.exp(d) / np.exp(d).sum()
    codes = rng.choice(k, (n, 1), p=q) if scored else np.full((n, 1), 2)
    target = np.broadcast_to(t, (n, 2, k))
    drafts = np.broadcast_to(d, (n, 1, k)) if scored else None
    accepted, out = Q.verify(target, 1.0, drafts, 1.0, codes, rng.random((n, 2)))
    p = np.exp(t) / np.exp(t).sum()
    share = np.bincount(out[:, 0], minlength=k) / n
    assert (np.abs(share - p) < 5 * np.sqrt(p * (1 - p) / n)).all()
    assert ((accepted == 1) == (out[:, 1] >= 0)).all()
