"""GPU: the rounding of the sums of a table's gradient does not grow with the number of a code's positions: through the C ABI, against exact sums."""
import numpy as np
import pytest

import scores_ref as R

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
# Additions behind one another on the way of a member to the sum of its code: for a group of lanes, which has 512 members at most, the first two, 64
# eights, three within an eight, seven that are no eight.  Sixteen groups that share 1024 have fewer: eight eights each, and sixteen sums; then, in
# 64 bits, the pieces.
DEPTH = 2 + 64 + 3 + 7


@pytest.fixture(scope="module")
def ctx():
    import vq_amd
    c = vq_amd.Context(0)
    yield c
    c.close()


def sums(ctx, g, codes, k, kind="f32"):
    n, dim = g.shape
    out = ctx.empty((k, dim), np.float32)
    ctx.code_embed_grad(kind, ctx.to_device(R.pack(g, kind)), n, dim, dim, 1, 4, ctx.to_device(codes.astype(np.int32)), 1, 1.0, k, False, "f32", out, dim)
    return out.download().astype(np.float64)


@pytest.mark.parametrize("members,named,k,dim", [(1000, 64, 262_144, 16), (1024, 100, 262_144, 5), (300, 128, 262_144, 40), (96, 10, 5000, 16), (1024, 1, 40, 20),
                                                 (1025, 30, 70, 16), (5000, 3, 9, 24)])
@pytest.mark.parametrize("kind", R.TYPES)
def test_small_numbers_beside_a_large_one(ctx, members, named, k, dim, kind):
    """The first codes have many positions each, in one workgroup as many such codes as fit it; the first position of each has a one and the others
    half a step of it, which added to it one by one are lost."""
    least = 2.0 ** -24  # (f16's smallest number)
    codes = np.repeat(np.arange(named), members)
    g = np.full((codes.size, dim), least)
    g[::members] = 1.0
    mixed = np.arange(named * members).reshape(named, members).T.reshape(-1)  # the codes' positions among one another
    got = sums(ctx, g[mixed], codes[mixed], k, kind)
    want = 1.0 + (members - 1) * least
    assert (np.abs(got[:named] - want) <= (DEPTH + 1) * U * want).all(), np.abs(got[:named] - want).max() / U
    assert (got[named:] == 0).all()


def test_many_pieces_of_one_code(ctx):
    """Two million positions of a code: 2049 pieces, the first with 2^20, the others with half a step of it each."""
    n, dim = 2_098_000, 4
    g = np.full((n, dim), 2.0 ** -14)
    g[0] = 2.0 ** 20
    got = sums(ctx, g, np.zeros(n, int), 1)
    want = 2.0 ** 20 + (n - 1) * 2.0 ** -14
    assert (np.abs(got[0] - want) <= (DEPTH + 1) * U * want).all()
