"""Plain 64-bit forms of the operators of models over codes, and the bounds on a kernel's rounding that their tests use."""
import numpy as np

import scores_ref as R

U24, HALF_STEP, LEAST = R.U24, R.HALF_STEP, R.LEAST
CODES = {1: np.uint8, 2: np.uint16, 4: np.int32}


def rounded(want, err, kind):
    """How far a result may be that is off by err before it is rounded to the type."""
    return err + 1.01 * HALF_STEP[kind] * (np.abs(want) + err) + LEAST[kind]


def embed(table, codes, scale):
    """table: (m, k, dim) in 64 bits, codes: (n, m).  (rows, how far before rounding): m sums and the product with the scale, rounded
    once each, on at most the sum of the magnitudes."""
    m, k, dim = table.shape
    n = codes.shape[0]
    y, size = np.zeros((n, dim)), np.zeros((n, dim))
    for s in range(m):
        named = (codes[:, s] >= 0) & (codes[:, s] < k)
        t = table[s, codes[named, s]]
        y[named] += t
        size[named] += np.abs(t)
    y[(codes >= k).any(axis=1)] = np.nan
    return scale * y, 1.01 * (m + 1) * U24 * abs(scale) * size


def depth(count):
    """Additions behind one another on the way of a member of `count` to their sum: up to 1024 members in a row at the most; beyond that a
    sixteenth of the 1024 of a piece and sixteen sums, then a sixteenth of the pieces and sixteen sums."""
    return np.where(count <= 1024, count, 64 + 16 + count // 16384 + 18) + 1


def embed_grad(g, codes, scale, k, old=None):
    """g: (n, dim) in 64 bits.  (gradient (m, k, dim), how far before rounding)."""
    n, m = codes.shape
    out, size, count = np.zeros((m, k, g.shape[1])), np.zeros((m, k, g.shape[1])), np.zeros((m, k, 1))
    for s in range(m):
        named = (codes[:, s] >= 0) & (codes[:, s] < k)
        np.add.at(out[s], codes[named, s], g[named])
        np.add.at(size[s], codes[named, s], np.abs(g[named]))
        np.add.at(count[s], codes[named, s], 1.0)
    err = (depth(count) + 1) * U24 * abs(scale) * size
    out = scale * out
    if old is not None:
        out = out + old
        err = err + U24 * np.abs(out)
    return out, 1.01 * err


def teacher(lp, code, k, rest, possible):
    """Per row: q (of each entry), log q, whether there is any alternative, whether one is no code or no number, and which codes are alternatives;
    r, what they leave (possible: a row has another code that can be)."""
    n, top = lp.shape
    has = (code >= 0) & ~(lp == -np.inf)
    with np.errstate(invalid="ignore", over="ignore"):
        bad = (has & ((code >= k) | ~(lp < np.inf))).any(axis=1)
    some = has.any(axis=1)
    l = np.where(has & ~bad[:, None], lp, -np.inf).astype(np.float64)
    if not rest:
        most = l.max(axis=1, keepdims=True)
        most = np.where(most == -np.inf, 0.0, most)
        total = np.exp(l - most).sum(axis=1, keepdims=True)
        with np.errstate(divide="ignore"):
            l = l - most - np.where(total > 0, np.log(np.where(total > 0, total, 1.0)), 0.0)
    q = np.exp(l)
    r = np.where(some & possible & ~bad, np.maximum(0.0, 1.0 - q.sum(axis=1)), 0.0) if rest else np.zeros(n)
    named = np.zeros((n, k), bool)
    i, t = np.nonzero(has & (code < k))
    named[i, code[i, t]] = True
    return dict(q=q, lq=l, some=some, bad=bad, named=named, r=r, has=has)


def distill(x, beta, lp, code, rest):
    """Of rows of scores in 64 bits: the loss, m, L and log R, and how far the kernel's may be (none for m)."""
    n, k = x.shape
    st = R.statistics(x, beta)
    tL, _ = R.bounds(st, k)
    named0 = teacher(lp, code, k, False, np.ones(n, bool))["named"]
    other = np.where(named0, -np.inf, x)
    with np.errstate(invalid="ignore", divide="ignore"):
        so = R.statistics(other, beta)
        tO, _ = R.bounds(so, k)
        dm = beta * (so["m"] - np.where(st["none"], 0.0, st["m"]))
        logrest = np.where(so["none"], -np.inf, dm + so["L"] - np.where(st["none"], 0.0, st["L"]))
        # the rest's own sum, the difference of the two largest scores (rounded three times) and L; with R apart, L is joined of two sums
        elr = 1.01 * (tO + tL + 4 * U24 * (np.abs(dm) + np.abs(so["L"]) + np.abs(st["L"]) + 1))
        logrest[st["bad"]] = np.nan
        tL = tL + 4 * U24 * (1 + st["A"])
        t = teacher(lp, code, k, rest, ~so["none"])
        c = np.clip(code, 0, k - 1)
        rows = np.arange(n)[:, None]
        logp = st["lp"][rows, c]
        d = np.abs(st["d"][rows, c])
        q = np.where(t["q"] > 2.0 ** -149, t["q"], 0.0)
        terms = np.where(q > 0, q * (t["lq"] - logp), 0.0)
        elq = 4 * U24 * (np.abs(lp) + np.abs(t["lq"]) + 1)
        elp = (2 * d + np.abs(logp)) * U24 * 1.01 + tL[:, None]
        # a product and a sum rounded per entry, q rounded once
        err = np.where(q > 0, q * (elq + elp) + 4 * U24 * np.abs(terms), 0.0).sum(axis=1) + 8 * U24 * np.abs(terms).sum(axis=1)
        loss = terms.sum(axis=1)
        r = t["r"]
        more = np.where(r > 0, r * (np.log(np.where(r > 0, r, 1.0)) - logrest), 0.0)
        err = err + np.where(r > 0, r * (elr + 4 * U24 * (np.abs(np.log(np.where(r > 0, r, 1.0))) + 1)) + 8 * U24 * np.abs(more), 0.0)
        loss = loss + more
    loss[st["none"] & t["some"]] = np.inf
    loss[st["bad"] | t["bad"]] = np.nan
    loss[~t["some"]] = 0.0
    return dict(loss=loss, m=st["m"], L=st["L"], logrest=logrest, none=st["none"], bad=st["bad"], tloss=1.01 * err + 2.0 ** -140, tL=tL, tlogrest=elr)


def distill_grad(x, beta, lp, code, rest, m, L, logrest, g):
    """(gradient, how far before rounding), from the statistics as they are given."""
    n, k = x.shape
    m, L = m.astype(np.float64), L.astype(np.float64)
    none, bad = m == -np.inf, np.isnan(L)
    lr = logrest.astype(np.float64) if rest else np.full(n, -np.inf)
    open_ = rest & (lr != -np.inf) & ~np.isnan(lr)
    t = teacher(lp, code, k, rest, open_)
    bad = bad | t["bad"]
    r, Q = t["r"], t["q"].sum(axis=1)
    total = (1.0 if not rest else Q + r) * np.ones(n)
    qc = np.zeros((n, k))
    i, j = np.nonzero(t["has"] & (code < k))
    np.add.at(qc, (i, code[i, j]), t["q"][i, j])
    with np.errstate(invalid="ignore", over="ignore"):
        d = beta * (x - np.where(none, 0.0, m)[:, None])
        logp = d - np.where(none, 0.0, L)[:, None]
        p = np.exp(logp)
        elp = np.where(p > 0, (4 * np.abs(np.where(p > 0, d, 0)) + 2 * np.abs(np.where(p > 0, logp, 0)) + 8 + 4 * np.abs(np.where(none, 0, L))[:, None]) * U24, 0.0)
        bg = (beta * g.astype(np.float64))[:, None]
        y = np.where(t["named"], bg * (total[:, None] * p - qc), bg * total[:, None] * p)
        err = np.abs(bg) * (p * total[:, None] * (elp + 8 * U24) + 8 * U24 * qc + 2.0 ** -126 * (1 + total[:, None]))
        if rest:
            lrs = np.where(open_, lr, 0.0)
            share = np.where(open_[:, None], np.exp(logp - lrs[:, None]), 0.0)
            factor = total * np.exp(lrs) - r
            yo = bg * share * factor[:, None]
            ef = (total * np.exp(lrs) * (4 + 2 * np.abs(lrs)) + r * 4) * U24 + 4 * U24 * np.abs(factor)
            eo = np.abs(bg) * (share * (ef[:, None] + np.abs(factor)[:, None] * (elp + 4 * U24 * (np.abs(lrs)[:, None] + 2))) + 2.0 ** -126 * (1 + np.abs(factor[:, None])))
            use = ~t["named"] & open_[:, None]
            y, err = np.where(use, yo, y), np.where(use, eo, err)
    err = err + 2.0 ** -149
    y[none] = 0.0
    y[bad] = np.nan
    y[~t["some"]] = 0.0
    return y, 1.01 * err


def _softmax(x, beta):
    m = x.max() if x.size else -np.inf
    if np.isnan(x).any() or m == np.inf or m == -np.inf:
        return None
    e = np.exp(beta * (x - m))
    return e / e.sum()


def verify(target, beta, drafts, beta_draft, codes, u):
    """target: (n, draft + 1, k), drafts: (n, draft, k) or None, in 64 bits; codes (n, draft), u (n, draft + 1).  (accepted, out)."""
    n, rows, k = target.shape
    draft = rows - 1
    accepted, out = np.zeros(n, np.int64), np.full((n, rows), -1, np.int64)
    for b in range(n):
        weights, a = None, 0
        while weights is None:
            p = _softmax(target[b, a], beta)
            if p is None:
                break
            if a == draft or codes[b, a] < 0:
                weights = p
                break
            c = codes[b, a]
            q = None
            if drafts is not None:
                q = _softmax(drafts[b, a], beta_draft)
                if q is None:
                    break
            if c >= k:
                break
            if u[b, a] * (1.0 if q is None else q[c]) < p[c]:
                out[b, a] = c
                a += 1
                continue
            if q is None:
                weights = p.copy()
                weights[c] = 0.0
            else:
                weights = np.maximum(p - q, 0.0)
                if weights.sum() == 0:
                    weights = p
        accepted[b] = a
        if weights is not None and weights.sum() > 0:
            cdf = np.cumsum(weights)
            over = np.nonzero((cdf > u[b, draft] * cdf[-1]) & (weights > 0))[0]
            out[b, a] = over[0] if over.size else np.nonzero(weights > 0)[0][-1]
    return accepted, out
