"""Plain 64-bit forms of the operators on rows of logits, and the bounds that
the tests hold the kernels to.

Bounds.  A weight 2^y, y = (l - m) * c in fp32, is off by 2^-22 (the
exponential's own error) and by 2^-22 ln 2 |y| (the difference, c and the
product, each rounded); a sum of weights by their mean error and by its own
roundings, of which no path to it has more than 64 (2^-24 each: 2^-18).  So the
sum is off by e_S = 2^-18 + 2^-22 + 2^-22 E with E = sum p |y| ln 2 at most.
Weights below 2^-126 are 0 in fp32 without subnormal numbers: as S is 1 or
more, a p is off by 2^-126 besides, and what it is multiplied by counts (the
weight over the temperature can be 1e10).
"""
import torch

HALF = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}     # a rounding, relative
LEAST = {torch.float32: 2.0 ** -126, torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -126}  # and at the low end


def fp32(v):
    """What passes fp32 is infinite there."""
    return v.float().double().where(v.float().isinf(), v)


def without(logits):
    """Rows that hold no distribution: NaN, +inf or only -inf."""
    x = logits.double()
    return x.isnan().any(1) | (x == float("inf")).any(1) | (x == -float("inf")).all(1)


def rows(logits, T):
    """ln p, p, m, S, and the bound e_S of each row (0 in rows without a distribution)."""
    logits = torch.where(without(logits)[:, None], torch.zeros_like(logits), logits)
    x = logits.double() / T
    lp = torch.log_softmax(x, 1)
    p = lp.exp()
    m = logits.double().amax(1)
    y = torch.where(p > 0, (m[:, None] / T - x).clamp(max=200.0), torch.zeros_like(x))
    return lp, p, m, (x - m[:, None] / T).exp().sum(1), 2.0 ** -18 + 2.0 ** -22 + 2.0 ** -22 * (p * y).sum(1)


def logprobs(logits, tokens, T, k):
    """(values, bounds): logp, entropy, rmax, rsum, and top_ids, top_logp."""
    lp, p, m, S, e = rows(logits, T)
    live = torch.ones_like(m, dtype=torch.bool) if tokens is None else (tokens >= 0) & (tokens < logits.shape[1])
    at = torch.zeros(len(m), 1, dtype=torch.int64) if tokens is None else tokens.clamp(0, logits.shape[1] - 1).long()[:, None]
    logp = lp.gather(1, at)[:, 0]
    ent = -torch.where(p > 0, p * lp, torch.zeros_like(p)).sum(1)
    # the entropy is ln S + sum p |y|: each of its sums is off by e_S, y itself by 2^-22
    val = [logp, ent, m, S]
    tol = [e + 2.0 ** -23 * logp.abs(), (e + 2.0 ** -22) * (2 + 2 * ent + S.log()), torch.zeros_like(m), (e + 2.0 ** -24) * S]
    none = without(logits)
    val = [torch.where(live, torch.where(none, torch.nan, fp32(v)), torch.zeros_like(v)) for v in val]
    tol = [torch.where(live, t, torch.zeros_like(t)) for t in tol]
    if k:
        ids = logits.float().sort(dim=1, descending=True, stable=True).indices[:, :k]
        top = lp.gather(1, ids)
        val += [torch.where((live & ~none)[:, None], ids, -1),
                torch.where(live[:, None], torch.where(none[:, None], torch.nan, fp32(top)), torch.zeros_like(top))]
        tol += [None, torch.where(live[:, None], e[:, None] + 2.0 ** -23 * top.abs(), torch.zeros_like(top))]
    return val, tol


def _rounded(val, off, dtype):
    """The bound of a value off by `off` that was rounded to dtype."""
    return off * (1 + 2 * HALF[dtype]) + HALF[dtype] * val.abs() + LEAST[dtype]


def logprobs_grad(logits, tokens, T, d_logp, d_entropy, dtype):
    """(dlogits, bound): each term of an element is off by its weight's error and by a few roundings."""
    lp, p, m, S, e = rows(logits, T)
    n, V = logits.shape
    ok = torch.ones(n, dtype=torch.bool) if tokens is None else (tokens >= 0) & (tokens < V)
    dl = torch.zeros(n, dtype=torch.float64) if d_logp is None else d_logp.double()
    de = torch.zeros(n, dtype=torch.float64) if d_entropy is None else d_entropy.double()
    ok = ok & ((dl != 0) | (de != 0))
    lpz = torch.where(p > 0, lp, torch.zeros_like(lp))
    H = -(p * lpz).sum(1)
    hot = torch.zeros_like(p)
    if d_logp is not None:
        hot.scatter_(1, tokens.clamp(0, V - 1).long()[:, None], 1.0)
    g = dl[:, None] * (hot - p) - de[:, None] * p * (lpz + H[:, None])
    # the weight, S and the entropy (given in fp32, off by (e + 2^-22)(2 + 2H + ln S)): 8 roundings besides
    y = (m[:, None] / T - logits.double() / T).clamp(max=200.0)
    rel = 2.0 ** -21 + 2.0 ** -22 * y + e[:, None]
    ent = (e + 2.0 ** -22) * (2 + 2 * H + S.log())
    off = p * (rel * (dl.abs()[:, None] + de.abs()[:, None] * (lpz.abs() + H[:, None] + S.log()[:, None] + y))
               + (de.abs() * ent)[:, None]) + 2.0 ** -22 * hot * dl.abs()[:, None]
    g, off = g / T, off / T
    g, off = torch.where(ok[:, None], g, torch.zeros_like(g)), torch.where(ok[:, None], off, torch.zeros_like(off))
    return g, _rounded(g, off, dtype)


def teacher(ids, t, V, T):
    """q of each entry (0 where it does not count, or below 2^-126) and whether the row has any."""
    has = (ids >= 0) & (ids < V) & (t > -float("inf"))
    live = has.any(1)
    s = t.double().masked_fill(~has, -float("inf")) / T
    q = torch.softmax(torch.where(live[:, None], s, torch.zeros_like(s)), 1)
    return torch.where(live[:, None] & has & (q >= 2.0 ** -126), q, torch.zeros_like(q)), live


def distill(logits, ids, t, T, weight, dtype):
    """(values, bounds): loss, rmax, rsum, dlogits (dtype None: without)."""
    lp, p, m, S, e = rows(logits, T)
    n, V = logits.shape
    q, live = teacher(ids, t, V, T)
    at = lp.gather(1, ids.clamp(0, V - 1).long())
    lq = torch.where(q > 0, q.log(), torch.zeros_like(q))
    terms = torch.where(q > 0, q * (lq - at), torch.zeros_like(q))
    loss = terms.sum(1)
    # a q is off by 2^-22 and 2^-23 |t| of itself, |t| <= -ln q: times the term; ln p by e_S; the result by a rounding
    size = torch.where(q > 0, q * (lq.abs() + at.abs()), torch.zeros_like(q)).nan_to_num(0.0, 0.0, 0.0)
    qrel = 2.0 ** -20 + 2.0 ** -22 * lq.abs()
    ltol = (size * qrel).sum(1) + e + 2.0 ** -24 * loss.abs()
    z = torch.zeros_like(m)
    val = [torch.where(live, fp32(v), z) for v in (loss, m, S)]
    tol = [torch.where(live, v, z) for v in (ltol, z, (e + 2.0 ** -24) * S)]
    if dtype is None:
        return val, tol
    w = torch.ones_like(m) if weight is None else weight.double()
    w = torch.where(live, w, z) / T
    places = torch.zeros_like(p).scatter_add_(1, ids.clamp(0, V - 1).long(), q)
    g = (p - places) * w[:, None]
    y = (m[:, None] / T - logits.double() / T).clamp(max=200.0)
    off = p * (2.0 ** -21 + 2.0 ** -22 * y + e[:, None]) + 2.0 ** -126 + torch.zeros_like(p).scatter_add_(1, ids.clamp(0, V - 1).long(), q * qrel)
    return val + [g], tol + [_rounded(g, off * w.abs()[:, None], dtype)]
