"""Plain 64-bit forms of the 8-bit scores and of the log probabilities of codes, and the bounds on a kernel's rounding
that the tests of both use."""
import numpy as np

U24 = 2.0 ** -24  # half a step of binary32, relative
HALF_STEP = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}
LEAST = {"f32": 2.0 ** -150, "f16": 2.0 ** -25, "bf16": 2.0 ** -134}  # half a step of the type's subnormal numbers
TYPES = ("f32", "f16", "bf16")


def pack(x, kind):
    """Values rounded to the type, as the array that is uploaded."""
    x = np.ascontiguousarray(x, np.float32)
    if kind == "f32":
        return x
    if kind == "f16":
        with np.errstate(over="ignore"):
            return x.astype(np.float16)
    u = x.view(np.uint32).astype(np.uint64)
    r = ((u + 0x7FFF + ((u >> 16) & 1)) >> 16).astype(np.uint16)
    return np.where(np.isnan(x), np.uint16(0x7FC0), r).astype(np.uint16)


def unpack(a, kind):
    """The values in 64 bits of an array of the type."""
    if kind == "bf16":
        return (a.astype(np.uint32) << 16).view(np.float32).astype(np.float64)
    return a.astype(np.float64)


def f32(x):
    """Rounded to binary32: -inf where a value is beyond its range, as a log probability of beta * -3.3e38, beta = 20, is."""
    with np.errstate(over="ignore"):
        return x.astype(np.float32)


def rows_i8(x):
    """(integers, scales) of rows in 64 bits: the scale is rounded to binary32, the quotient by it is exact enough
    (53 bits) to tell a tie from its neighbours."""
    with np.errstate(invalid="ignore"):
        s = (np.abs(x).max(axis=1) / 127.0).astype(np.float32)
    bad = ~np.isfinite(x).all(axis=1)
    s[bad] = np.nan
    d = s.astype(np.float64)[:, None]
    with np.errstate(invalid="ignore", divide="ignore"):
        q = np.rint(x / d)
    q[(s == 0) | bad] = 0
    return np.clip(q, -127, 127).astype(np.int8), s


def scores(xq, xs, wq, ws, bias, kind):
    """(scores, how far a kernel's may be): the sum is exact; its conversion, two products and the sum with the bias are
    rounded once each, then the result to its type."""
    y0 = (xq.astype(np.float64) @ wq.astype(np.float64).T) * xs.astype(np.float64)[:, None] * ws.astype(np.float64)
    y = y0 + (0.0 if bias is None else bias.astype(np.float64))
    err = 3.01 * U24 * np.abs(y0) + U24 * np.abs(y)
    return y, err + 1.01 * HALF_STEP[kind] * (np.abs(y) + err) + LEAST[kind]


def statistics(x, beta):
    """Of rows of scores in 64 bits: m, L, H, log p (rows of -inf and rows with NaN or +inf as the header says)."""
    m = x.max(axis=1) if x.size else np.zeros(0)
    none = m == -np.inf
    with np.errstate(invalid="ignore", divide="ignore", over="ignore"):
        d = beta * (x - np.where(none, 0.0, m)[:, None])
        e = np.exp(d)
        S = e.sum(axis=1)
        L = np.log(S)
        A = -np.where(e > 0, d * e, 0.0).sum(axis=1) / S
        Q = np.where(e > 0, d * d * e, 0.0).sum(axis=1) / S
        H = np.where(none, 0.0, L + A)
        lp = d - np.where(none, 0.0, L)[:, None]
    bad = np.isnan(S)
    H[bad] = np.nan
    lp[bad] = np.nan
    lp[none] = -np.inf
    return dict(m=m, L=L, H=H, lp=lp, A=np.where(none, 0.0, A), Q=np.where(none, 0.0, Q), none=none, bad=bad, d=d)


def bounds(st, k):
    """How far L and H of a kernel in 32 bits may be.  An exponent beta * (x - m) is rounded twice and multiplied by
    log2 e (two more): 4 |d| of 2^-24; the exponential is within 4 of them; a lane adds at most k / 128 + 64 terms before
    sums are joined, each sum rounded.  Averaged with the weights p: sum p |d| = A, sum p d^2 = Q."""
    depth = min(k, k // 128 + 64) + 8
    with np.errstate(invalid="ignore"):
        L = (4 * st["A"] + 4 + depth) * U24 + 2 * U24 * np.abs(st["L"])
        H = L + (4 * st["Q"] + (8 + 2 * depth) * st["A"]) * U24 + 2 * U24 * np.abs(st["H"])
    return 1.01 * L, 1.01 * H


def best(x, top):
    """Codes of the largest scores, of equal ones the lower code first; -1 behind the last one above -inf."""
    n, k = x.shape
    at = np.argsort(-(x + 0.0), axis=1, kind="stable")[:, :top]
    out = np.full((n, top), -1, np.int64)
    for i in range(n):
        for t in range(min(top, k)):
            if x[i, at[i, t]] > -np.inf:
                out[i, t] = at[i, t]
    return out


def grad(x, beta, codes, m, L, H, gl, gh):
    """(gradient in 64 bits, how far a kernel's may be before its result is rounded to the type), from the statistics as
    they are given.  log p: 4 |d| and |log p| of 2^-24; p: that, and 4; log p + H and the products: 4 more.  A probability below
    2^-126, the smallest normal number, may count as zero: it is off by at most as much, and the gradient by beta times its factor."""
    n, k = x.shape
    none, bad = m == -np.inf, np.isnan(L)
    gl = np.zeros(n) if gl is None else gl.astype(np.float64)
    H = np.zeros(n) if gh is None else H.astype(np.float64)
    gh = np.zeros(n) if gh is None else gh.astype(np.float64)
    gl = np.where(codes < 0, 0.0, np.where(codes >= k, np.nan, gl))
    with np.errstate(invalid="ignore", over="ignore"):
        d = beta * (x - np.where(none, 0.0, m.astype(np.float64))[:, None])
        lp = d - np.where(none, 0.0, L.astype(np.float64))[:, None]
        p = np.exp(lp)
        lpz = np.where(p > 0, lp, 0.0)
        dz = np.where(p > 0, d, 0.0)
        one = np.arange(k) == codes[:, None]
        inner = gl[:, None] + gh[:, None] * (lpz + H[:, None])
        g = beta * (np.where(one, gl[:, None], 0.0) - np.where(p > 0, p * inner, 0.0))
        elp = (4 * np.abs(dz) + 2 * np.abs(lpz)) * U24
        size = np.abs(gl)[:, None] + np.abs(gh)[:, None] * (np.abs(lpz) + np.abs(H)[:, None])
        err = beta * p * (size * (elp + 8 * U24) + np.abs(gh)[:, None] * elp) + 4 * U24 * np.abs(g) + beta * size * 2.0 ** -126 + 2.0 ** -149
    g[none] = 0.0
    err[none] = 0.0
    g[bad] = np.nan
    return g, 1.01 * err
