"""Performance cases of the 8-bit scores and of the log probabilities of codes.

A program that models codes (those of a trained codebook, or any vocabulary of k codes) scores rows
against k codewords and reads probabilities from the scores.  The operators, as `vq_amd.Context` has
them, on rows that lie in GPU memory:

  scores     8-bit rows times 8-bit codewords, a scale per row and per codeword, a bias per codeword
  rows       floating rows to 8-bit rows with a scale each, then their scores
  logprobs   log probability of a given code per row, entropy, and the best alternatives, from scores
  grad       the gradient of a loss over log probabilities and entropies with respect to the scores

With `own` false, `run` computes the same from elementary torch operations.
"""
import math

import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
BYTES = {"f32": 4, "f16": 2, "bf16": 2}


def listed():
    return [
        # one row against the codewords of a byte: latency only
        dict(name="scores_one", op="scores", n=1, dim=128, k=256, out="f32", bias=True, pad=True),
        # a step of a server with 16 rows in flight against the largest code range: the codebook's bytes count
        dict(name="scores_serve", op="scores", n=16, dim=1280, k=65536, out="bf16", bias=False, pad=True),
        # odd everything: rows, components and codes
        dict(name="scores_ragged", op="scores", n=4099, dim=1000, k=777, out="f16", bias=True, pad=True),
        # a large batch through a wide layer: the matrix rate counts; the largest case
        dict(name="scores_large", op="scores", n=16384, dim=8192, k=8192, out="bf16", bias=False, pad=True),
        # a small batch of embeddings as it arrives, quantized and scored
        dict(name="rows_small", op="rows", n=32, dim=768, k=1024, type="f32", out="f32", bias=True),
        # a million rows of the headline width against one codebook: the scores' own bytes count
        dict(name="rows_1m", op="rows", n=1_000_000, dim=128, k=256, type="bf16", out="f32", bias=True),
        # one row of a model's answer over the largest code range
        dict(name="logprobs_one", op="logprobs", n=1, k=65536, type="f32", top=20, beta=1.0, codes=4, masked=0.0, empty=0, pad=0),
        # byte codes of a million rows of scores, and the second-best code of each
        dict(name="logprobs_1m", op="logprobs", n=1_000_000, k=256, type="f32", top=2, beta=0.5, codes=1, masked=0.0, empty=0, pad=0),
        # answers under a mask of allowed codes, some rows with none left; padded rows of an odd number of codes
        dict(name="logprobs_masked", op="logprobs", n=777, k=50_021, type="f16", top=5, beta=1.25, codes=4, masked=0.3, empty=5, pad=27),
        # scoring a batch of sequences over the largest code range
        dict(name="logprobs_batch", op="logprobs", n=8192, k=65536, type="bf16", top=8, beta=1.0, codes=2, masked=0.0, empty=0, pad=0),
        # the backward pass of a small batch, odd numbers of rows and codes
        dict(name="grad_small", op="grad", n=333, k=1001, type="f32", beta=0.7, codes=4, masked=0.1, empty=2, pad=0),
        # the backward pass of a batch of sequences over the largest code range
        dict(name="grad_batch", op="grad", n=8192, k=65536, type="bf16", beta=1.0, codes=2, masked=0.0, empty=0, pad=0),
    ]


def _log(rng, lo, hi):
    """A whole number between lo and hi, spread over the logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["scores", "scores", "rows", "logprobs", "logprobs", "grad"])
    if op in ("scores", "rows"):
        # an odd size as often as one that tiles divide
        step = rng.choice([1, 1, 64])
        dim = max(16, _log(rng, 16, 8192) // step * step)
        k = max(2, _log(rng, 16, 65536) // step * step)
        most = max(1, min(1_000_000, 2 ** 28 // k, 2 ** 28 // dim, 2 ** 40 // (dim * k)))
        c = dict(op=op, n=_log(rng, 1, most), dim=dim, k=k, out=rng.choice(["f32", "f16", "bf16"]), bias=rng.random() < 0.5)
        c.update(dict(pad=rng.random() < 0.8) if op == "scores" else dict(type=rng.choice(["f32", "f16", "bf16"])))
        return c
    kind = rng.choice(["f32", "f16", "bf16"])
    k = _log(rng, 16, 262_144)
    c = dict(op=op, n=_log(rng, 1, min(1_000_000, 2 ** 28 // k)), k=k, type=kind, beta=rng.choice([1.0, 0.5, 1.5]),
             codes=rng.choice([4] + [2] * (k <= 65536) + [1] * (k <= 256)), masked=rng.choice([0.0, 0.0, 0.4]), pad=rng.choice([0, 0, 5, 64]))
    c["empty"] = rng.choice([0, 3]) if c["n"] > 8 else 0
    if op == "logprobs":
        c["top"] = rng.choice([0, 1, 5, 20, 32])
    return c


# ---- inputs ----------------------------------------------------------------------------------------
_kept = {}


def _context():
    """The one context that a program keeps."""
    if "ctx" not in _kept:
        import vq_amd
        _kept["ctx"] = vq_amd.Context(0)
    return _kept["ctx"]


def _stride(dim, pad):
    """Bytes from one 8-bit row to the next: padded to 16, or the rows one after the other."""
    return (dim + 15) // 16 * 16 if pad else dim


def _bytes_of(n, dim, ld, g):
    """8-bit rows as a quantizer leaves them: values up to 127, one of them at the end of the range; what lies
    between the rows is not zero."""
    q = torch.randn((n, ld), generator=g, device="cuda").mul_(40).round_().clamp_(-127, 127).to(torch.int8)
    q[:, 0] = 127
    return q


def prepare(case, seed):
    c = dict(case)
    g = torch.Generator(device="cuda").manual_seed(seed)
    op, n, k = c["op"], c["n"], c["k"]
    s = dict(case=c)
    if op in ("scores", "rows"):
        dim = c["dim"]
        pad = c.get("pad", True)
        s["ld"] = ld = _stride(dim, pad)
        s["w"] = _bytes_of(k, dim, ld, g)
        s["ws"] = torch.rand((k,), generator=g, device="cuda").mul_(0.01).add_(0.005)
        s["bias"] = torch.randn((k,), generator=g, device="cuda") if c["bias"] else None
        if op == "scores":
            s["x"] = _bytes_of(n, dim, ld, g)
            s["xs"] = torch.rand((n,), generator=g, device="cuda").mul_(0.01).add_(0.005)
        else:
            rows = torch.randn((n, dim), generator=g, device="cuda")
            # rows of different lengths, as embeddings have them
            s["rows"] = rows.mul_(torch.rand((n, 1), generator=g, device="cuda").add_(0.5)).to(TYPES[c["type"]])
            s["x"] = torch.empty((n, ld), dtype=torch.int8, device="cuda")
            s["xs"] = torch.empty((n,), device="cuda")
        s["out"] = torch.empty((n, k), dtype=TYPES[c["out"]], device="cuda")
        return s
    ld = s["ld"] = k + c["pad"]
    x = torch.randn((n, ld), generator=g, device="cuda").mul_(2.5)
    codes = torch.randint(0, k, (n,), generator=g, device="cuda")
    if c["masked"]:
        gone = torch.rand((n, ld), generator=g, device="cuda") < c["masked"]
        x[gone] = -math.inf
    if c["empty"]:
        x[torch.arange(c["empty"], device="cuda") * (n // c["empty"])] = -math.inf
    s["scores"] = x.to(TYPES[c["type"]])
    del x
    if c["codes"] == 4 and n > 4:
        codes[n // 3] = -1  # a row of the batch without a code
    s["codes"] = codes.to({1: torch.uint8, 2: torch.uint16, 4: torch.int32}[c["codes"]])
    if op == "logprobs":
        top = c["top"]
        s["logprob"], s["max"], s["logsum"], s["entropy"] = (torch.empty((n,), device="cuda") for _ in range(4))
        s["top_logprob"] = torch.empty((n, top), device="cuda")
        s["top_code"] = torch.empty((n, top), dtype=torch.int32, device="cuda")
        return s
    # what the forward pass left, and the loss's gradients: a weight per row, and a reward for entropy
    s["max"], s["logsum"], s["entropy"] = (torch.cat(v) for v in zip(
        *(_statistics(r.float(), c["beta"]) for r in s["scores"][:, :k].split(max(1, 2 ** 26 // k)))))
    s["g_logprob"] = torch.randn((n,), generator=g, device="cuda")
    s["g_entropy"] = torch.rand((n,), generator=g, device="cuda").mul_(0.1)
    s["out"] = torch.empty((n, ld), dtype=s["scores"].dtype, device="cuda")[:, :k]
    return s


# ---- plain forms -----------------------------------------------------------------------------------
def _statistics(x, beta):
    """Largest score, log of the sum of exponentials relative to it, and entropy of softmax(beta x), by rows."""
    m = x.amax(1)
    none = m == -math.inf
    d = (x - m.masked_fill(none, 0.0)[:, None]).mul_(beta)
    e = d.exp()
    total = e.sum(1)
    logsum = total.log()
    d.masked_fill_(e == 0, 0.0)
    entropy = logsum - d.mul_(e).sum(1) / total
    return m, logsum, entropy.masked_fill(none, 0.0)


def _at_codes(x, m, logsum, codes, beta):
    """log p of one code per row: 0 where a row has none, NaN where its code is none of the k."""
    c = codes.to(torch.int64)
    v = x.gather(1, c.clamp(0, x.shape[1] - 1)[:, None])[:, 0]
    lp = (v - m.masked_fill(m == -math.inf, 0.0)) * beta - logsum.masked_fill(logsum == -math.inf, 0.0)
    return lp.masked_fill(c >= x.shape[1], math.nan).masked_fill(c < 0, 0.0)


def _plain_logprobs(s):
    c = s["case"]
    k, top, beta = c["k"], c["top"], c["beta"]
    x = s["scores"][:, :k].float()
    m, logsum, entropy = _statistics(x, beta)
    lp = _at_codes(x, m, logsum, s["codes"], beta)
    if not top:
        return lp, m, logsum, entropy
    v, at = x.sort(dim=1, descending=True, stable=True)
    v, at = v[:, :top], at[:, :top]
    if top > k:
        v = torch.nn.functional.pad(v, (0, top - k), value=-math.inf)
        at = torch.nn.functional.pad(at, (0, top - k))
    none = v == -math.inf
    tl = (v - m[:, None]) * beta - logsum[:, None]
    return lp, m, logsum, entropy, tl.masked_fill(none, -math.inf), at.masked_fill(none, -1).to(torch.int32)


def _plain_grad(s):
    c = s["case"]
    k, beta = c["k"], c["beta"]
    none = s["max"] == -math.inf
    logp = (s["scores"][:, :k].float() - s["max"].masked_fill(none, 0.0)[:, None]).mul_(beta)
    logp.sub_(s["logsum"].masked_fill(none, 0.0)[:, None])
    p = logp.exp()
    codes = s["codes"].to(torch.int64)
    g = torch.where(codes < 0, 0.0, s["g_logprob"])
    logp.masked_fill_(p == 0, 0.0)
    out = p * (logp.add_(s["entropy"][:, None]).mul_(-s["g_entropy"][:, None]) - g[:, None])
    out.scatter_add_(1, codes.clamp(min=0)[:, None], g[:, None])
    return (out * beta).masked_fill(none[:, None], 0.0).to(s["scores"].dtype)


def _plain_scores(x, xs, s):
    c = s["case"]
    y = (x[:, :c["dim"]].float() @ s["w"][:, :c["dim"]].float().T).mul_(xs[:, None]).mul_(s["ws"])
    if s["bias"] is not None:
        y.add_(s["bias"])
    return y.to(TYPES[c["out"]])


def _plain_rows(x):
    """8-bit rows and their scales; the quotients in 64 bits, for values next to the border of two integers."""
    scale = (x.abs().amax(1).double() / 127).float()
    return (x.double() / scale.double()[:, None]).round_().nan_to_num_(0.0), scale


def run(state):
    s, c = state, state["case"]
    op, n, k = c["op"], c["n"], c["k"]
    if not own:
        if op == "scores":
            return _plain_scores(s["x"], s["xs"], s)
        if op == "rows":
            q, scale = _plain_rows(s["rows"])
            return _plain_scores(q, scale, s), scale
        return _plain_logprobs(s) if op == "logprobs" else _plain_grad(s)
    ctx = _context()
    if op in ("scores", "rows"):
        dim, ld, out = c["dim"], s["ld"], s["out"]
        if op == "rows":
            ctx.rows_i8(c["type"], s["rows"].data_ptr(), n, dim, dim, s["x"].data_ptr(), ld, s["xs"].data_ptr())
        ctx.scores_i8(s["x"].data_ptr(), s["xs"].data_ptr(), n, ld, s["w"].data_ptr(), s["ws"].data_ptr(), k, ld, dim,
                      s["bias"].data_ptr() if c["bias"] else None, c["out"], out.data_ptr(), k)
        return out if op == "scores" else (out, s["xs"])
    if op == "logprobs":
        top = c["top"]
        ctx.code_logprobs(c["type"], s["scores"].data_ptr(), n, s["ld"], k, c["beta"], c["codes"], s["codes"].data_ptr(), 1,
                          top, s["logprob"].data_ptr(), s["max"].data_ptr(), s["logsum"].data_ptr(), s["entropy"].data_ptr(),
                          s["top_logprob"].data_ptr() if top else None, s["top_code"].data_ptr() if top else None)
        got = s["logprob"], s["max"], s["logsum"], s["entropy"]
        return got + (s["top_logprob"], s["top_code"]) if top else got
    ctx.code_logprobs_grad(c["type"], s["scores"].data_ptr(), n, s["ld"], k, c["beta"], c["codes"], s["codes"].data_ptr(), 1,
                           s["max"].data_ptr(), s["logsum"].data_ptr(), s["entropy"].data_ptr(), s["g_logprob"].data_ptr(),
                           s["g_entropy"].data_ptr(), s["out"].data_ptr(), s["ld"])
    return s["out"]


# ---- what a pass cannot do without -----------------------------------------------------------------
def work(case):
    c = case
    op, n, k = c["op"], c["n"], c["k"]
    if op in ("scores", "rows"):
        dim = c["dim"]
        rows = n * dim * (1 if op == "scores" else BYTES[c["type"]]) + 4 * n
        return {"bytes": float(rows + k * dim + 4 * k * (2 if c["bias"] else 1) + n * k * BYTES[c["out"]]), "flops": 2.0 * n * k * dim}
    e = BYTES[c["type"]]
    if op == "logprobs":
        return {"bytes": float(n * (k * e + c["codes"] + 16 + 8 * c["top"])), "flops": 5.0 * n * k}
    return {"bytes": float(n * (2 * k * e + c["codes"] + 20)), "flops": 8.0 * n * k}


# ---- the definitions in 64 bits --------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    c = s["case"]
    op, k = c["op"], c["k"]
    if op in ("scores", "rows"):
        if 2.0 * c["n"] * k * c["dim"] > 3e12:
            return None
        d = c["dim"]
        if op == "scores":
            q, scale = s["x"][:, :d].double(), s["xs"].double()
        else:
            # the scale is what the call hands out, a 32-bit number; the integer is the nearest to the quotient by it
            scale = (s["rows"].double().abs().max(dim=1).values / 127).float().double()
            q = torch.round(s["rows"].double() / scale[:, None])
        y = torch.matmul(q, s["w"][:, :d].double().t()) * (scale[:, None] * s["ws"].double()[None, :])
        if c["bias"]:
            y = y + s["bias"].double()
        return y if op == "scores" else (y, scale)
    beta = c["beta"]
    if op == "logprobs":
        parts = [_exact_logprobs(x, cd, beta, c["top"]) for x, cd in zip(s["scores"][:, :k].split(max(1, 2 ** 26 // k)),
                                                                         s["codes"].split(max(1, 2 ** 26 // k)))]
        return tuple(torch.cat(p) for p in zip(*parts))
    z = s["scores"][:, :k].double() * beta
    left = ~torch.isneginf(z).all(dim=1)
    p = torch.softmax(z, dim=1)
    plogp = torch.special.xlogy(p, p)
    h = -plogp.sum(dim=1, keepdim=True)
    code = s["codes"].long()
    has = code >= 0
    gl = torch.where(has, s["g_logprob"].double(), torch.zeros_like(z[:, 0]))
    grad = -gl[:, None] * p - s["g_entropy"].double()[:, None] * (plogp + p * h)
    rows = torch.arange(z.shape[0], device=z.device)[has]
    grad[rows, code[has]] += gl[has]
    grad *= beta
    grad[~left] = 0.0
    return grad


def _exact_logprobs(x, codes, beta, top):
    z = x.double() * beta
    left = ~torch.isneginf(z).all(dim=1)
    lse = torch.logsumexp(z, dim=1)
    m = x.double().max(dim=1).values
    logsum = torch.where(left, lse - m * beta, lse)
    p = torch.softmax(z, dim=1)
    h = torch.where(left, -torch.special.xlogy(p, p).sum(dim=1), torch.zeros_like(lse))
    code = codes.long()
    at = z[torch.arange(z.shape[0], device=z.device), code.clamp(min=0)]
    lp = torch.where(code < 0, torch.zeros_like(at), torch.where(left, at - lse, at))
    if not top:
        return lp, m, logsum, h
    t = min(top, x.shape[1])
    best = z.topk(t, dim=1).values
    best = torch.cat([best, best.new_full((best.shape[0], top - t), -math.inf)], dim=1)
    best = torch.where(torch.isneginf(best), best, best - lse[:, None])
    return lp, m, logsum, h, best
