"""GPU: drafted codes and the code that comes next where scores lie so far below their row's largest that a code has no weight."""
import numpy as np
import pytest

import scores_ref as R

pytestmark = pytest.mark.gpu
LN2 = float(np.log(2.0))


@pytest.fixture(scope="module")
def ctx():
    import vq_amd
    c = vq_amd.Context(0)
    yield c
    c.close()


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("n", [1, 3, 1100])  # the last one: four parts of a row to a workgroup
@pytest.mark.parametrize("scored", [None, False, True])
def test_the_first_code_with_a_weight(ctx, kind, n, scored):
    """Codes 2^-1050 below the largest count as none, also where those after them, 2^-550 below, lie in the same workgroup's parts: a random
    number of zero takes the first code with a weight.  By drawing, behind drafts without scores and with them."""
    k, part = 16384 + 100, 4096
    row = np.zeros(k)
    row[:part], row[part:16384] = -1050 * LN2, -550 * LN2
    row = R.unpack(R.pack(row, kind), kind)
    draft = 0 if scored is None else 1
    x = np.tile(row, (n * (draft + 1), 1))
    dx = ctx.to_device(R.pack(x, kind))
    u = np.zeros((n, draft + 1), np.float32)
    u[::2, :draft] = 0.999  # every second sequence's draft does not stay: q is 1, or next to it, and p a hundredth
    codes = np.full((n, 1), 16384 + 7, np.int32)
    dd = None
    if scored:  # the drafts' scores: the row's but that their own code has nearly all, so that p - q leaves the others'
        d = np.tile(row, (n, 1))
        d[:, 16384 + 7] = 64.0
        dd = ctx.to_device(R.pack(d, kind))
    accepted, out = ctx.empty(n, np.int32), ctx.empty((n, draft + 1), np.int32)
    ctx.code_verify(kind, dx, k, 1.0, dd, k, 1.0, n, draft, k, 4, ctx.to_device(codes) if draft else None, 1, ctx.to_device(u), draft + 1, accepted, out, draft + 1)
    a, o = accepted.download(), out.download()
    if draft:
        assert (a == np.arange(n) % 2).all()
        assert (o[1::2] == [16384 + 7, part]).all()
        assert (o[::2] == [part, -1]).all()
    else:
        assert (a == 0).all() and (o == part).all()
