"""Performance cases of what a model over codes reads, learns from and answers with.

A model whose alphabet are the k codes of a codebook (or of the m codebooks of a residual quantizer) reads codes through a
table of vectors, may learn from a larger model's best alternatives, and answers faster where a small model's drafts are
verified.  The operators, as `vq_amd.Context` has them, on arrays that lie in GPU memory:

  embed       the sum of a table's rows that a position's codes name, times a scale
  embed_grad  the gradient of the table's rows, from that of the sums
  distill     a row of scores against a teacher's best alternatives: the loss, and its gradient in the same call
  back        that gradient alone, from what the loss's call left
  verify      drafted codes against the model's probabilities, with given random numbers, and the code that comes next

With `own` false, `run` computes the same from elementary torch operations.
"""
import math

import numpy as np
import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
BYTES = {"f32": 4, "f16": 2, "bf16": 2}
CODES = {1: torch.uint8, 2: torch.uint16, 4: torch.int32}


def listed():
    return [
        # a step of a server with 16 rows in flight, from the largest code range: latency only
        dict(name="embed_step", op="embed", n=16, m=1, k=65536, dim=1280, type="bf16", out="bf16", codes=4, skew=True, none=0.0, pad=0),
        # sequences of a residual quantizer's codes, eight stages each: the rows that the codes name count
        dict(name="embed_stages", op="embed", n=65536, m=8, k=1024, dim=1024, type="bf16", out="bf16", codes=2, skew=False, none=0.0, pad=0),
        # the backward pass of a small padded batch, odd numbers of everything
        dict(name="embed_grad_small", op="embed_grad", n=333, m=1, k=1001, dim=100, type="f32", out="f32", codes=4, skew=True, none=0.1, pad=3),
        # a batch of sequences whose codes are as uneven as words are: the gradient's own bytes count
        dict(name="embed_grad_batch", op="embed_grad", n=16384, m=1, k=65536, dim=1280, type="bf16", out="f32", codes=4, skew=True, none=0.05, pad=0),
        # byte codes of a million rows of the headline width: every row of the table has thousands of members
        dict(name="embed_grad_1m", op="embed_grad", n=1_000_000, m=1, k=256, dim=128, type="bf16", out="f32", codes=1, skew=False, none=0.0, pad=0),
        # a training step's loss and gradient on a small batch, odd numbers of rows and codes
        dict(name="distill_small", op="distill", n=333, k=1001, type="f32", beta=0.5, top=5, rest=False, grad=True, masked=0.0, empty=0, pad=0),
        # loss and gradient of a batch of sequences over the largest code range
        dict(name="distill_batch", op="distill", n=8192, k=65536, type="bf16", beta=1.0, top=20, rest=False, grad=True, masked=0.0, empty=0, pad=0),
        # the loss alone, under a mask of allowed codes, what the alternatives leave as one more class; padded rows
        dict(name="distill_masked", op="distill", n=777, k=50_021, type="f16", beta=1.25, top=32, rest=True, grad=False, masked=0.3, empty=5, pad=27),
        # the backward pass alone, where the loss's own gradient came later
        dict(name="distill_back", op="back", n=2048, k=65536, type="f32", beta=1.0, top=16, rest=True, masked=0.0, empty=0, pad=0),
        # one user's answer, four codes drafted: latency
        dict(name="verify_one", op="verify", n=1, draft=4, k=65536, type="f32", beta=1.0, beta_draft=1.0, codes=4, greedy=False, masked=0.0, ragged=False, pad=0),
        # drafts looked up in the text so far, of different lengths; allowed codes only, an odd number of them
        dict(name="verify_ragged", op="verify", n=61, draft=3, k=50_021, type="f16", beta=1.25, beta_draft=1.0, codes=4, greedy=True, masked=0.3, ragged=True, pad=27),
        # a server's batch with a drafting model
        dict(name="verify_batch", op="verify", n=128, draft=5, k=65536, type="bf16", beta=1.0, beta_draft=0.8, codes=2, greedy=False, masked=0.0, ragged=False, pad=0),
    ]


def _log(rng, lo, hi):
    """A whole number between lo and hi, spread over the logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["embed", "embed_grad", "embed_grad", "distill", "distill", "back", "verify", "verify"])
    step = rng.choice([1, 1, 64])  # an odd size as often as one that tiles divide
    if op in ("embed", "embed_grad"):
        dim = max(16, _log(rng, 16, 4096) // step * step)
        m = rng.choice([1, 1, 2, 4, 8])
        k = max(16, min(_log(rng, 16, 262_144), 2 ** 27 // (dim * m)) // step * step)
        c = dict(op=op, n=_log(rng, 1, max(1, min(1_000_000, 2 ** 28 // (dim * m)))), m=m, k=k, dim=dim, type=rng.choice(list(TYPES)), out=rng.choice(list(TYPES)),
                 codes=rng.choice([4] + [2] * (k <= 65536) + [1] * (k <= 256)), skew=rng.random() < 0.5, pad=rng.choice([0, 0, 3, 64]))
        c["none"] = rng.choice([0.0, 0.1]) if c["codes"] == 4 else 0.0
        return c
    k = max(16, _log(rng, 16, 262_144) // step * step)
    c = dict(op=op, k=k, type=rng.choice(list(TYPES)), beta=rng.choice([1.0, 0.5, 1.5]), masked=rng.choice([0.0, 0.0, 0.4]), pad=rng.choice([0, 0, 5, 64]))
    if op == "verify":
        c.update(draft=rng.choice([0, 1, 3, 4, 8]), beta_draft=rng.choice([1.0, 0.7]), greedy=rng.random() < 0.3, ragged=rng.random() < 0.3,
                 codes=rng.choice([4] + [2] * (k <= 65536) + [1] * (k <= 256)))
        c["ragged"] = c["ragged"] and c["codes"] == 4
        c["n"] = _log(rng, 1, max(1, min(512, 2 ** 25 // (k * (c["draft"] + 1)))))
        return c
    c.update(n=_log(rng, 1, min(100_000, 2 ** 28 // k)), top=rng.choice([1, 5, 20, 32, 64]), rest=rng.random() < 0.5)
    c["empty"] = rng.choice([0, 3]) if c["n"] > 8 else 0
    if op == "distill":
        c["grad"] = rng.random() < 0.6
    return c


# ---- inputs ----------------------------------------------------------------------------------------
_kept = {}


def _context():
    """The one context that a program keeps."""
    if "ctx" not in _kept:
        import vq_amd
        _kept["ctx"] = vq_amd.Context(0)
    return _kept["ctx"]


def _draw_codes(c, g):
    """n * m codes; skewed ones as uneven as words are, the j-th most frequent of k with a probability near 1 / (j ln k)."""
    n, m, k = c["n"], c["m"], c["k"]
    if not c["skew"]:
        return torch.randint(0, k, (n, m), generator=g, device="cuda")
    u = torch.rand((n, m), generator=g, device="cuda", dtype=torch.float64)
    rank = ((u * math.log(k + 1)).exp() - 1).long().clamp_(0, k - 1)
    return torch.randperm(k, generator=g, device="cuda")[rank]


def _distinct(n, k, skew):
    """How many of k codes n drawn ones hold, on average."""
    if not skew:
        return k * -math.expm1(n * math.log1p(-1.0 / k))
    p = np.log1p(1.0 / np.arange(1, k + 1)) / math.log(k + 1)
    return float(-np.expm1(n * np.log1p(-p)).sum())


def _rows(n, k, pad, masked, g, kind, spread=2.5):
    """Rows of scores, a share of them masked."""
    x = torch.randn((n, k + pad), generator=g, device="cuda").mul_(spread)
    gone = None
    if masked:
        gone = torch.rand((n, k + pad), generator=g, device="cuda") < masked
        gone[:, 0] = False
        x[gone] = -math.inf
    return x.to(TYPES[kind]), gone


def _prepare_embed(c, g):
    n, m, k, dim = c["n"], c["m"], c["k"], c["dim"]
    codes = _draw_codes(c, g)
    if c["none"]:
        codes[torch.rand((n, m), generator=g, device="cuda") < c["none"]] = -1
    s = dict(case=c, codes=codes.to(CODES[c["codes"]]), ld=dim + c["pad"])
    if c["op"] == "embed":
        s["scale"] = math.sqrt(dim)
        s["table"] = torch.randn((m * k, s["ld"]), generator=g, device="cuda").mul_(0.02).to(TYPES[c["type"]])
        s["out"] = torch.empty((n, dim), dtype=TYPES[c["out"]], device="cuda")
    else:
        s["scale"] = math.sqrt(dim)
        s["rows"] = torch.randn((n, s["ld"]), generator=g, device="cuda").mul_(0.01).to(TYPES[c["type"]])
        s["grad"] = torch.empty((m * k, dim), dtype=TYPES[c["out"]], device="cuda")
    return s


def _prepare_distill(c, g):
    n, k, top = c["n"], c["k"], c["top"]
    x, _ = _rows(n, k, c["pad"], c["masked"], g, c["type"])
    s = dict(case=c, ld=k + c["pad"])
    # a teacher that sees much the same as its student, and more sharply; where the student's mask rules a code out, so does the teacher's
    lp = torch.empty((n, top), device="cuda").fill_(-math.inf)
    code = torch.empty((n, top), dtype=torch.int32, device="cuda").fill_(-1)
    t = min(top, k)
    at = 0
    for part in x[:, :k].split(max(1, 2 ** 26 // k)):
        y = (part.float() * 1.2).add_(torch.randn(part.shape, generator=g, device="cuda"))
        best, where = torch.log_softmax(y * c["beta"], 1).topk(t, dim=1)
        r = slice(at, at + part.shape[0])
        lp[r, :t] = best
        code[r, :t] = torch.where(best == -math.inf, -1, where).to(torch.int32)
        at += part.shape[0]
    short = torch.arange(n, device="cuda") % 97 == 5  # shorter lists, as a filter of unlikely codes leaves them
    lp[short, (top + 1) // 2:] = -math.inf
    code[short, (top + 1) // 2:] = -1
    if c["empty"]:  # padded positions: no teacher, and nothing that may be answered
        rows = torch.arange(c["empty"], device="cuda") * (n // c["empty"])
        x[rows], lp[rows], code[rows] = -math.inf, -math.inf, -1
    s.update(scores=x, lp=lp, code=code)
    s["loss"], s["max"], s["logsum"], s["logrest"] = (torch.empty((n,), device="cuda") for _ in range(4))
    if c["op"] == "back":
        parts = [_row_statistics(r.float(), a, b, c["beta"])[:3] for r, a, b in zip(
            *(v.split(max(1, 2 ** 26 // k)) for v in (x[:, :k], lp, code)))]
        s["max"], s["logsum"], s["logrest"] = (torch.cat(v) for v in zip(*parts))
    if c["op"] == "back" or c["grad"]:
        s["g"] = torch.rand((n,), generator=g, device="cuda").add_(0.5)  # a weight per row
        s["grad"] = torch.empty((n, s["ld"]), dtype=x.dtype, device="cuda")[:, :k]
    return s


def _prepare_verify(c, g):
    n, d, k = c["n"], c["draft"], c["k"]
    x, gone = _rows(n * (d + 1), k, c["pad"], c["masked"], g, c["type"], 3.0)
    s = dict(case=c, ld=k + c["pad"], target=x, draft=None)
    s["uniform"] = torch.rand((n, d + 1), generator=g, device="cuda")
    s["accepted"] = torch.empty((n,), dtype=torch.int32, device="cuda")
    s["out"] = torch.empty((n, d + 1), dtype=torch.int32, device="cuda")
    s["codes"] = None
    if not d:
        return s
    seen = x.view(n, d + 1, -1)[:, :d].reshape(n * d, -1)
    y = seen.float() + torch.randn(seen.shape, generator=g, device="cuda")
    y = y.to(TYPES[c["type"]])
    if c["greedy"]:
        codes = y[:, :k].float().argmax(1)
    else:
        s["draft"] = y
        codes = torch.cat([torch.multinomial(torch.softmax(p.float() * c["beta_draft"], 1), 1, generator=g)[:, 0] for p in y[:, :k].split(256)])
    codes = codes.view(n, d)
    if c["ragged"]:
        length = torch.randint(0, d + 1, (n, 1), generator=g, device="cuda")
        codes[torch.arange(d, device="cuda")[None, :] >= length] = -1
    s["codes"] = codes.to(CODES[c["codes"]])
    return s


def prepare(case, seed):
    c = dict(case)
    g = torch.Generator(device="cuda").manual_seed(seed)
    if c["op"] in ("embed", "embed_grad"):
        return _prepare_embed(c, g)
    return _prepare_verify(c, g) if c["op"] == "verify" else _prepare_distill(c, g)


# ---- plain forms -----------------------------------------------------------------------------------
def _plain_embed(s):
    c = s["case"]
    codes = s["codes"].to(torch.int64)
    y = torch.zeros((c["n"], c["dim"]), device="cuda")
    for i in range(c["m"]):
        code = codes[:, i]
        y.add_(s["table"][code.clamp(min=0) + i * c["k"], :c["dim"]].float().masked_fill_((code < 0)[:, None], 0.0))
    return y.mul_(s["scale"]).to(TYPES[c["out"]])


def _plain_embed_grad(s):
    """Sums by code in 64 bits: a code may have many thousands of members."""
    c = s["case"]
    codes, rows = s["codes"].to(torch.int64), s["rows"][:, :c["dim"]].double()
    y = torch.zeros((c["m"] * c["k"] + 1, c["dim"]), device="cuda", dtype=torch.float64)
    for i in range(c["m"]):
        code = codes[:, i]
        y.index_add_(0, torch.where(code < 0, c["m"] * c["k"], code + i * c["k"]), rows)
    return y[:-1].mul_(s["scale"]).to(TYPES[c["out"]])


def _row_statistics(x, lp, code, beta):
    """Of rows of scores: the largest, the log of the sum of exponentials relative to it, the log of the share of the
    codes that are no alternative, and which codes are (a column more holds what is none)."""
    n, k = x.shape
    m = x.amax(1)
    none = m == -math.inf
    e = (x - m.masked_fill(none, 0.0)[:, None]).mul_(beta).exp_()
    logsum = e.sum(1).log()
    named = torch.zeros((n, k + 1), dtype=torch.bool, device=x.device)
    named.scatter_(1, torch.where((code >= 0) & (lp > -math.inf), code.long(), k), True)
    named = named[:, :k]
    # relative to the largest of the rest: its share may be far below the smallest number
    rest = x.masked_fill(named, -math.inf)
    mr = rest.amax(1)
    gone = mr == -math.inf
    sr = (rest - mr.masked_fill(gone, 0.0)[:, None]).mul_(beta).exp_().sum(1)
    logrest = (mr - m.masked_fill(none, 0.0)) * beta + sr.log() - logsum.masked_fill(none, 0.0)
    return m, logsum, logrest.masked_fill(gone, -math.inf), named


def _teacher(lp, code, rest, logrest):
    """Probabilities and log probabilities of the teacher's alternatives, and of what they leave, which is the small
    difference of one and their sum: in 64 bits."""
    lp = lp.double().masked_fill(code < 0, -math.inf)
    if not rest:
        top = lp.amax(1, keepdim=True)
        top = top.masked_fill(top == -math.inf, 0.0)
        total = (lp - top).exp().sum(1, keepdim=True)
        lp = lp - top - total.log().masked_fill(total == 0, 0.0)
    q = lp.exp()
    r = torch.zeros_like(q[:, 0])
    if rest:
        listed_any = (q > 0).any(1)
        r = torch.where(listed_any & (logrest > -math.inf), (1.0 - q.sum(1)).clamp(min=0.0), 0.0)
    return q.float(), lp.float(), r.float()


def _plain_distill(s):
    c = s["case"]
    beta, code, k = c["beta"], s["code"].long(), c["k"]
    x = s["scores"][:, :k].float()
    if c["op"] == "back":
        m, logsum, logrest = s["max"], s["logsum"], s["logrest"]
        named = torch.zeros((c["n"], k + 1), dtype=torch.bool, device="cuda")
        named = named.scatter_(1, torch.where((code >= 0) & (s["lp"] > -math.inf), code, k), True)[:, :k]
    else:
        m, logsum, logrest, named = _row_statistics(x, s["lp"], s["code"], beta)
    none = m == -math.inf
    q, lq, r = _teacher(s["lp"], s["code"], c["rest"], logrest)
    out = []
    if c["op"] == "distill":
        mine = (x.gather(1, code.clamp(min=0)) - m.masked_fill(none, 0.0)[:, None]) * beta - logsum.masked_fill(none, 0.0)[:, None]
        loss = torch.where(q > 0, q * (lq - mine), 0.0).sum(1)
        if c["rest"]:
            loss = loss + torch.where(r > 0, r * (r.log() - logrest), 0.0)
        out = [loss, m, logsum] + [logrest] * c["rest"]
        if not c["grad"]:
            return tuple(out)
    p = (x - m.masked_fill(none, 0.0)[:, None]).mul_(beta).sub_(logsum.masked_fill(none, 0.0)[:, None])
    total = q.sum(1) + r
    if c["rest"]:
        # codes that are no alternative: their share of the rest, times what the rest has above the teacher's
        share = (p - logrest.masked_fill(logrest == -math.inf, 0.0)[:, None]).exp_().mul_((total * logrest.exp() - r)[:, None])
        p = torch.where(named, p.exp_().mul_(total[:, None]), share)
    else:
        p = p.exp_().mul_(total[:, None])
    p.scatter_add_(1, code.clamp(min=0), -q)
    p.mul_((s["g"] * beta)[:, None]).masked_fill_(none[:, None], 0.0)
    out.append(p.to(s["scores"].dtype))
    return tuple(out) if len(out) > 1 else out[0]


def _softmax64(x, beta):
    z = x.double() * beta
    z = (z - z.amax(-1, keepdim=True)).exp_()
    return z / z.sum(-1, keepdim=True)


def _plain_verify(s):
    """In 64 bits: which code comes next hangs on sums next to one another."""
    c = s["case"]
    n, d, k = c["n"], c["draft"], c["k"]
    u = s["uniform"].double()
    p = _softmax64(s["target"][:, :k], c["beta"]).view(n, d + 1, k)
    accepted = torch.zeros((n,), dtype=torch.int64, device="cuda")
    each = torch.arange(n, device="cuda")
    if d:
        codes = s["codes"].to(torch.int64)
        has = (codes >= 0).long().cumprod(1).bool()
        at = codes.clamp(min=0)[:, :, None]
        if c["greedy"]:
            qc = torch.ones((n, d), dtype=torch.float64, device="cuda")
        else:
            q = _softmax64(s["draft"][:, :k], c["beta_draft"]).view(n, d, k)
            qc = q.gather(2, at)[:, :, 0]
        ok = has & (u[:, :d] * qc < p[:, :d].gather(2, at)[:, :, 0])
        accepted = ok.long().cumprod(1).sum(1)
        refused = accepted < has.sum(1)
        pos = accepted.clamp(max=d - 1)
        w = p[each, accepted]
        if c["greedy"]:
            w.scatter_(1, codes[each, pos].clamp(min=0)[:, None], torch.where(refused, 0.0, w.gather(1, codes[each, pos].clamp(min=0)[:, None])[:, 0])[:, None])
        else:
            w = torch.where(refused[:, None], (w - q[each, pos]).clamp(min=0.0), w)
    else:
        w = p[:, 0]
    cdf = w.cumsum(1)
    nxt = (cdf <= (u[:, d] * cdf[:, -1])[:, None]).sum(1)
    out = torch.full((n, d + 1), -1, dtype=torch.int64, device="cuda")
    if d:
        out[:, :d] = torch.where(torch.arange(d, device="cuda")[None, :] < accepted[:, None], codes, -1)
    out[each, accepted] = nxt
    return accepted.to(torch.int32), out.to(torch.int32)


def run(state):
    s, c = state, state["case"]
    op, n, k = c["op"], c["n"], c["k"]
    if not own:
        if op == "embed":
            return _plain_embed(s)
        if op == "embed_grad":
            return _plain_embed_grad(s)
        return _plain_verify(s) if op == "verify" else _plain_distill(s)
    ctx = _context()
    if op == "embed":
        ctx.code_embed(c["type"], s["table"].data_ptr(), k, s["ld"], c["dim"], c["m"], c["codes"], s["codes"].data_ptr(), n, c["m"],
                       s["scale"], c["out"], s["out"].data_ptr(), c["dim"])
        return s["out"]
    if op == "embed_grad":
        ctx.code_embed_grad(c["type"], s["rows"].data_ptr(), n, s["ld"], c["dim"], c["m"], c["codes"], s["codes"].data_ptr(), c["m"],
                            s["scale"], k, False, c["out"], s["grad"].data_ptr(), c["dim"])
        return s["grad"]
    if op == "distill":
        with_grad = c["grad"]
        ctx.code_distill(c["type"], s["scores"].data_ptr(), n, s["ld"], k, c["beta"], c["top"], s["lp"].data_ptr(), s["code"].data_ptr(), c["top"],
                         c["rest"], s["loss"].data_ptr(), s["max"].data_ptr(), s["logsum"].data_ptr(), s["logrest"].data_ptr() if c["rest"] else None,
                         s["g"].data_ptr() if with_grad else None, s["grad"].data_ptr() if with_grad else None, s["ld"])
        got = (s["loss"], s["max"], s["logsum"]) + ((s["logrest"],) if c["rest"] else ())
        return got + (s["grad"],) if with_grad else got
    if op == "back":
        ctx.code_distill_grad(c["type"], s["scores"].data_ptr(), n, s["ld"], k, c["beta"], c["top"], s["lp"].data_ptr(), s["code"].data_ptr(), c["top"],
                              c["rest"], s["max"].data_ptr(), s["logsum"].data_ptr(), s["logrest"].data_ptr() if c["rest"] else None, s["g"].data_ptr(),
                              s["grad"].data_ptr(), s["ld"])
        return s["grad"]
    ctx.code_verify(c["type"], s["target"].data_ptr(), s["ld"], c["beta"], s["draft"].data_ptr() if s["draft"] is not None else None, s["ld"],
                    c["beta_draft"], n, c["draft"], k, c["codes"], s["codes"].data_ptr() if c["draft"] else None, max(1, c["draft"]),
                    s["uniform"].data_ptr(), c["draft"] + 1, s["accepted"].data_ptr(), s["out"].data_ptr(), c["draft"] + 1)
    return s["accepted"], s["out"]


# ---- what a pass cannot do without -----------------------------------------------------------------
def work(case):
    c = case
    op, n, k = c["op"], c["n"], c["k"]
    if op in ("embed", "embed_grad"):
        m, dim = c["m"], c["dim"]
        if op == "embed":
            size = m * _distinct(n, k, c["skew"]) * dim * BYTES[c["type"]] + n * dim * BYTES[c["out"]]
        else:
            size = n * dim * BYTES[c["type"]] + m * k * dim * BYTES[c["out"]]
        return {"bytes": float(size + n * m * c["codes"]), "flops": float(n * m * dim)}
    e = BYTES[c["type"]]
    if op == "verify":
        rows = n * (c["draft"] + 1) + (0 if c["greedy"] else n * c["draft"])
        return {"bytes": float(rows * k * e + n * (c["draft"] * (c["codes"] + 8) + 16)), "flops": 4.0 * rows * k}
    lists = n * (c["top"] * 8 + 16 + 4 * c["rest"])
    if op == "back":
        return {"bytes": float(2 * n * k * e + lists), "flops": 4.0 * n * k}
    return {"bytes": float((2 if c["grad"] else 1) * n * k * e + lists), "flops": (8.0 if c["grad"] else 4.0) * n * k}


# ---- the definitions in 64 bits --------------------------------------------------------------------
def _exact_embed(s):
    c = s["case"]
    n, m, k, dim = c["n"], c["m"], c["k"], c["dim"]
    code = s["codes"].long()
    if c["op"] == "embed":
        out = torch.zeros((n, dim), dtype=torch.float64, device="cuda")
        for i in range(m):
            named = code[:, i] >= 0
            out[named] += s["table"][i * k + code[named, i], :dim].double()
        return out * s["scale"]
    out = torch.zeros((m, k, dim), dtype=torch.float64, device="cuda")
    for i in range(m):
        named = torch.nonzero(code[:, i] >= 0)[:, 0]
        order = torch.argsort(code[named, i], stable=True)
        for rows in named[order].split(1 << 18):  # the members of a code lie side by side
            out[i].index_add_(0, code[rows, i], s["rows"][rows, :dim].double())
    return (out * s["scale"]).view(m * k, dim)


def _exact_rows(c, x, lp, code, g, stats):
    """Loss and what else the case returns, for some rows.  stats: what a separate backward pass is given, or None."""
    n, k = x.shape
    z = x.double() * c["beta"]
    lse = torch.logsumexp(z, 1)
    dead = torch.isneginf(lse)
    valid = (code >= 0) & ~torch.isneginf(lp)
    idx = torch.where(valid, code.long(), 0)
    t = torch.where(valid, lp.double(), torch.full_like(lp, -math.inf, dtype=torch.float64))
    some = valid.any(1)
    count = torch.zeros((n, k), dtype=torch.float64, device=x.device).scatter_add_(1, idx, valid.double())
    lse_rest = torch.logsumexp(torch.where(count > 0, torch.full_like(z, -math.inf), z), 1)
    logrest = torch.where(torch.isneginf(lse_rest), lse_rest, lse_rest - lse)
    given = stats is not None
    if given:  # the gradient is that of the given statistics
        m32, L32, R32 = (v.double() for v in stats)
        lse = torch.where(dead, lse, m32 * c["beta"] + L32)
        logrest = R32
    if c["rest"]:
        q = t.exp()
        r = torch.where(some & ~torch.isneginf(logrest), (1.0 - q.sum(1)).clamp(min=0.0), torch.zeros_like(lse))
    else:
        norm = torch.logsumexp(t, 1, keepdim=True)
        t = torch.where(some[:, None], t - norm, t)
        q, r = t.exp(), torch.zeros_like(lse)
    safe = torch.where(dead, torch.zeros_like(lse), lse)
    logp = z - safe[:, None]
    out = []
    if c["op"] == "distill":
        loss = (torch.special.xlogy(q, q) - torch.where(q > 0, q * logp.gather(1, idx), torch.zeros_like(q))).sum(1)
        loss = loss + torch.special.xlogy(r, r) - torch.where(r > 0, r * logrest, torch.zeros_like(r))
        m = x.double().max(1).values
        out = [loss, m, torch.where(dead, lse, lse - m * c["beta"])] + [logrest] * c["rest"]
        if not c["grad"]:
            return out
    p = logp.exp()
    mass = q.sum(1) + r
    d = p * mass[:, None]
    d.scatter_add_(1, idx, -q)
    if c["rest"]:
        inside = torch.where(torch.isneginf(logrest)[:, None], p * 0, (logp - torch.where(torch.isneginf(logrest), safe * 0, logrest)[:, None]).exp())
        d = torch.where(count > 0, d, inside * (mass * logrest.exp() - r)[:, None])
    d = d * (g.double() * c["beta"])[:, None]
    d[dead] = 0.0
    return out + [d]


def _exact_distill(s):
    c = s["case"]
    k = c["k"]
    parts = [s["scores"][:, :k], s["lp"], s["code"]]
    back = c["op"] == "back"
    with_grad = back or c["grad"]
    extra = [s["g"] if with_grad else s["loss"]] + ([s["max"], s["logsum"], s["logrest"]] if back else [])
    got = []
    for rows in zip(*(v.split(max(1, 2 ** 25 // k)) for v in parts + extra)):
        got.append(_exact_rows(c, rows[0], rows[1], rows[2], rows[3], rows[4:] if back else None))
    got = tuple(torch.cat(v) for v in zip(*got))
    return got if len(got) > 1 else got[0]


def _exact_verify(s):
    """A sequence at a time, in the log domain."""
    c = s["case"]
    n, d, k = c["n"], c["draft"], c["k"]
    target = s["target"].view(n, d + 1, -1)[:, :, :k]
    draft = s["draft"].view(n, d, -1)[:, :, :k] if s["draft"] is not None else None
    codes = s["codes"].to(torch.int64).tolist() if d else [[]] * n
    u = s["uniform"].double().tolist()
    accepted, out = [], []
    for b in range(n):
        row, a, weights = [], 0, None
        lp = torch.log_softmax(target[b].double() * c["beta"], 1)
        lq = torch.log_softmax(draft[b].double() * c["beta_draft"], 1) if draft is not None else None
        for pos, code in enumerate(codes[b]):
            if code < 0:
                break
            ratio = lp[pos, code].exp().item() / (1.0 if lq is None else lq[pos, code].exp().item())
            if u[b][pos] < ratio:
                row.append(code)
                a += 1
                continue
            weights = lp[pos].exp()
            if lq is None:
                weights[code] = 0.0
            else:
                weights = (weights - lq[pos].exp()).clamp(min=0.0)
            break
        if weights is None:
            weights = lp[a].exp()
        cdf = torch.cumsum(weights, 0)
        row.append(int(torch.searchsorted(cdf, cdf[-1:] * u[b][d], right=True).item()))
        accepted.append(a)
        out.append(row + [-1] * (d + 1 - len(row)))
    return torch.tensor(accepted, dtype=torch.int32, device="cuda"), torch.tensor(out, dtype=torch.int32, device="cuda").view(n, d + 1)


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] in ("embed", "embed_grad"):
        return _exact_embed(s)
    return _exact_verify(s) if case["op"] == "verify" else _exact_distill(s)
