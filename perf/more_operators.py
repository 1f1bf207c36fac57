"""Measured cases of the operators on rows of logits: log-probabilities of
given tokens with entropy and top alternatives, distillation from a teacher's
top logits, and the gradients of both.

Shapes: the vocabulary is the LM head's (262144), those of the framework's
tests, or generic; rows are single tokens, batches of them, and the tokens of a
training step.

A row holds logits l[0 .. vocab-1]; p = softmax(l / temperature).

logprobs       ln p of the row's token, the entropy -sum p ln p, the k largest
               logits' places (the lowest of several alike first) and ln p;
               also the row's largest logit m and S = sum exp((l - m) / T),
               from which p = exp((l - m) / T) / S.  A row whose token is
               negative is left out: zeros, places -1.
logprobs_grad  dl of sum_i d_logp[i] ln p(token i) + d_entropy[i] entropy[i]
distill        q = softmax(teacher / T) over the row's entries (places ids, -1
               where there are fewer); loss = sum q (ln q - ln p); and with
               the rows' weights the gradient (weight / T) (p - q).  A row
               without entries has loss 0 and gradient 0.
distill_grad   that gradient from m and S
"""
import math
import random

import torch

own = False

DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


# --------------------------------------------------------------------------
# cases
# --------------------------------------------------------------------------
def listed():
    return [
        # one decode step of one user who asked for alternatives (launch latency)
        dict(name="logp_decode_1", op="logprobs", rows=1, vocab=262144, x="f32", k=20, temperature=1.0, left=0, tail=0),
        # a serving batch, an odd vocabulary: rows off a 16-byte boundary
        dict(name="logp_decode_48", op="logprobs", rows=48, vocab=50257, x="f32", k=5, temperature=0.7, left=0, tail=0),
        # a training step's tokens scored under a model, fp32 logits as tk_linear_fwd writes them (bandwidth)
        dict(name="logp_score", op="logprobs", rows=4095, vocab=262144, x="f32", k=0, temperature=1.0, left=10, tail=0),
        # a teacher's pass over a batch: its 128 likeliest tokens are kept for distillation
        dict(name="logp_teacher", op="logprobs", rows=1024, vocab=262144, x="bf16", k=128, temperature=1.0, left=0, tail=0),
        # policy gradient with an entropy bonus over the answers' tokens; the prompts' are left out
        dict(name="policy_grad", op="logprobs_grad", rows=2048, vocab=131072, x="bf16", d="bf16", temperature=1.0, left=30,
             tail=0),
        # a few rows, fp32 gradients, an odd vocabulary
        dict(name="policy_grad_small", op="logprobs_grad", rows=33, vocab=32001, x="f32", d="f32", temperature=1.3, left=0,
             tail=0),
        # a distillation step over the tokens of a batch, loss and gradient in one call
        dict(name="distill_step", op="distill", rows=4096, vocab=262144, x="bf16", d="bf16", k=64, temperature=2.0, left=5,
             tail=0),
        # fp32 logits, bf16 gradients for tk_linear_dx; teacher lists of different length
        dict(name="distill_mixed", op="distill", rows=512, vocab=262144, x="f32", d="bf16", k=20, temperature=1.0, left=10,
             tail=144),
        # a small batch, an odd vocabulary
        dict(name="distill_small", op="distill", rows=16, vocab=50257, x="f16", d="f16", k=128, temperature=1.0, left=0,
             tail=0),
        # the loss alone, on held-out text
        dict(name="distill_loss", op="distill", rows=300, vocab=131072, x="f32", d=None, k=50, temperature=1.0, left=0, tail=0),
        # the backward pass of its own, when the loss's weights come later
        dict(name="distill_grad", op="distill_grad", rows=2048, vocab=262144, x="bf16", d="bf16", k=32, temperature=1.0, left=0,
             tail=0),
        # the same, a few fp32 rows of an odd vocabulary
        dict(name="distill_grad_odd", op="distill_grad", rows=100, vocab=50257, x="f32", d="f32", k=100, temperature=3.0,
             left=5, tail=0),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("logprobs", "logprobs", "logprobs_grad", "distill", "distill", "distill_grad"))
    vocab = _log(rng, 500, 262144)
    rows = _log(rng, 1, min(8192, (1 << 29) // vocab))
    case = dict(op=op, rows=rows, vocab=vocab, x=rng.choice(("f32", "f16", "bf16")),
                temperature=rng.choice((1.0, 1.0, 0.6, 1.7, 3.0)), left=rng.choice((0, 0, rng.randint(1, 60))),
                tail=rng.choice((0, 0, rng.randint(1, vocab // 8))))
    if op in ("logprobs", "distill", "distill_grad"):
        case["k"] = _log(rng, 1, 256)
    if op == "logprobs" and rng.random() < 0.4:
        case["k"] = 0
    if op != "logprobs":
        case["d"] = rng.choice((case["x"], case["x"], "f32", "bf16"))
    if op == "distill" and rng.random() < 0.25:
        case["d"] = None
    return case


def left_out(case):
    """Which rows have no token (no teacher entries): `left` in a hundred, spread over the batch."""
    return [(i * 61 + 17) % 100 < case["left"] for i in range(case["rows"])]


def work(case):
    live = case["rows"] - sum(left_out(case))
    size = lambda t: {"f32": 4, "f16": 2, "bf16": 2, None: 0}[t]  # noqa: E731
    logits, dl, k = live * case["vocab"] * size(case["x"]), case["rows"] * case["vocab"] * size(case.get("d")), case.get("k", 0)
    # (an exponential counts as one operation)
    if case["op"] == "logprobs":
        return {"bytes": float(logits + case["rows"] * (20 + 8 * k)), "flops": 7.0 * live * case["vocab"]}
    if case["op"] == "logprobs_grad":
        return {"bytes": float(logits + dl + case["rows"] * 24), "flops": 7.0 * live * case["vocab"]}
    passes = 2 if case["op"] == "distill" and case["d"] else 1
    return {"bytes": float(logits + dl + case["rows"] * (16 + 8 * k)), "flops": 5.0 * passes * live * case["vocab"]}


# --------------------------------------------------------------------------
# states
# --------------------------------------------------------------------------
_ctx = None


def _framework():
    global _ctx
    import tier_b200 as tk
    if _ctx is None:
        _ctx = tk.Context(torch.cuda.current_device())
    return tk, _ctx


def _blocks(n, vocab):
    """Rows in blocks of about 2^28 logits (the 64-bit forms and the inputs, to bound what they hold)."""
    step = max(1, (1 << 28) // vocab)
    return [slice(a, min(n, a + step)) for a in range(0, n, step)]


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    n, V, T = case["rows"], case["vocab"], case["temperature"]
    rand = lambda *s: torch.rand(*s, generator=g, device="cuda")  # noqa: E731
    left = torch.tensor(left_out(case), device="cuda")
    # a trained model's rows: a few likely tokens above a wide tail; a vocabulary padded to a rounder size ends in -inf
    some = min(32, V)
    top = torch.randint(V, (n, some), generator=g, device="cuda")
    above = 6.0 + 4.0 * rand(n, some)
    x = torch.empty(n, V, dtype=DT[case["x"]], device="cuda")
    for b in _blocks(n, V):
        t = torch.randn(b.stop - b.start, V, generator=g, device="cuda") * 2.0
        t.scatter_add_(1, top[b], above[b])
        if case["tail"]:
            t[:, V - case["tail"]:] = -math.inf
        x[b] = t.to(x.dtype)
    inside = V - case["tail"]
    # rows share a step's loss evenly; fp16 gradients come with a scaled loss, which keeps them out of its subnormals
    share = 1024.0 if case.get("d") == "f16" else 1.0 / n
    st = {"case": case, "x": x, "n": n}
    f32 = lambda *s: torch.zeros(*s, device="cuda")  # noqa: E731
    if "k" in case and case["op"] != "logprobs":
        # the teacher's list: its likeliest tokens, best first; some lists end early
        k = case["k"]
        ids, best = torch.zeros(n, k, dtype=torch.int64, device="cuda"), f32(n, k)
        for b in _blocks(n, V):
            t = x[b].float() + 0.7 * torch.randn(b.stop - b.start, V, generator=g, device="cuda")
            best[b], ids[b] = t.topk(k, dim=1)
        short = (rand(n, 1) < 0.2) & (torch.arange(k, device="cuda")[None] >= 1 + (rand(n, 1) * k).long())
        st["ids"] = torch.where(short | left[:, None], -1, ids).to(torch.int32)
        st["teacher"] = best
        st["weight"] = (0.5 + rand(n)) * share
    else:
        tokens = torch.where(rand(n) < 0.8, top[:, 0].clamp(max=inside - 1), torch.randint(inside, (n,), generator=g,
                                                                                           device="cuda"))
        st["tokens"] = torch.where(left, -1, tokens).to(torch.int32)
    if case["op"].endswith("_grad"):        # what the forward pass left
        st["rmax"], st["rsum"], st["entropy"] = f32(n), f32(n), f32(n)
        for b in _blocks(n, V):
            y = x[b].float()
            m = y.amax(1, keepdim=True)
            y = y.sub(m).div_(T).clamp_(min=-200.0)
            e = y.exp()
            s = e.sum(1, dtype=torch.float64)
            st["rmax"][b], st["rsum"][b] = m[:, 0], s.float()
            st["entropy"][b] = (s.log() - e.mul_(y).sum(1, dtype=torch.float64) / s).float()
        if case["op"] == "logprobs_grad":
            st["d_logp"] = torch.randn(n, generator=g, device="cuda") * share
            st["d_entropy"] = torch.full((n,), 0.01 * share, device="cuda")
    else:
        st["rmax"], st["rsum"] = f32(n), f32(n)
        if case["op"] == "logprobs":
            st["logp"], st["entropy"] = f32(n), f32(n)
            if case["k"]:
                st["top_ids"], st["top_logp"] = torch.zeros(n, case["k"], dtype=torch.int32, device="cuda"), f32(n, case["k"])
        else:
            st["loss"] = f32(n)
    if case.get("d"):
        st["dx"] = torch.zeros(n, V, dtype=DT[case["d"]], device="cuda")
    return st


# --------------------------------------------------------------------------
# one pass
# --------------------------------------------------------------------------
def run(st):
    case = st["case"]
    if own:
        return _run_own(st, case)
    return {"logprobs": _logprobs, "logprobs_grad": _logprobs_grad, "distill": _distill, "distill_grad": _distill_grad}[
        case["op"]](st, case)


def _run_own(st, case):
    tk, ctx = _framework()
    code = {"f32": tk.DT_F32, "f16": tk.DT_F16, "bf16": tk.DT_BF16}
    xt, T = code[case["x"]], case["temperature"]
    if case["op"] == "logprobs":
        ctx.logprobs(st["x"], st["tokens"], st["logp"], entropy=st["entropy"], rmax=st["rmax"], rsum=st["rsum"],
                     top_ids=st.get("top_ids"), top_logp=st.get("top_logp"), temperature=T, x_dtype=xt)
        res = (st["logp"], st["entropy"], st["rmax"], st["rsum"])
        return res + ((st["top_ids"], st["top_logp"]) if case["k"] else ())
    if case["op"] == "logprobs_grad":
        ctx.logprobs_grad(st["x"], st["tokens"], st["rmax"], st["rsum"], st["dx"], d_logp=st["d_logp"], entropy=st["entropy"],
                          d_entropy=st["d_entropy"], temperature=T, x_dtype=xt, d_dtype=code[case["d"]])
        return st["dx"]
    if case["op"] == "distill":
        grad = {"weight": st["weight"], "dlogits": st["dx"], "d_dtype": code[case["d"]]} if case["d"] else {}
        ctx.distill(st["x"], st["ids"], st["teacher"], st["loss"], rmax=st["rmax"], rsum=st["rsum"], temperature=T, x_dtype=xt,
                    **grad)
        return (st["loss"], st["rmax"], st["rsum"]) + ((st["dx"],) if case["d"] else ())
    ctx.distill_grad(st["x"], st["ids"], st["teacher"], st["rmax"], st["rsum"], st["dx"], weight=st["weight"], temperature=T,
                     x_dtype=xt, d_dtype=code[case["d"]])
    return st["dx"]


def _stats(st, T):
    """y = (l - m) / T, no lower than -200 (exp is 0 there), m, exp(y) and S."""
    x = st["x"].float()
    m = x.amax(1, keepdim=True)
    y = x.sub(m).div_(T).clamp_(min=-200.0)
    e = y.exp()
    return y, m, e, e.sum(1, keepdim=True)


def _logprobs(st, case):
    x, n, T = st["x"], st["n"], case["temperature"]
    y, m, e, s = _stats(st, T)
    live = st["tokens"] >= 0
    zero = torch.zeros(n, device="cuda")
    logp = torch.where(live, (y.gather(1, st["tokens"].clamp(min=0).long()[:, None]) - s.log())[:, 0], zero)
    entropy = torch.where(live, s.log()[:, 0] - e.mul_(y).sum(1) / s[:, 0], zero)
    res = (logp, entropy, torch.where(live, m[:, 0], zero), torch.where(live, s[:, 0], zero))
    if not case["k"]:
        return res
    del e
    k = min(case["k"], case["vocab"])
    ids = torch.zeros(n, k, dtype=torch.int64, device="cuda")
    for b in _blocks(n, case["vocab"]):
        ids[b] = x[b].float().sort(dim=1, descending=True, stable=True).indices[:, :k]
    lp = (x.gather(1, ids).float() - m) / T - s.log()
    return res + (torch.where(live[:, None], ids, -1).to(torch.int32), torch.where(live[:, None], lp, zero[:, None]))


def _given(st, T):
    """y and p from the forward pass's m and S."""
    y = st["x"].float().sub(st["rmax"][:, None]).div_(T).clamp_(min=-200.0)
    return y, y.exp() / st["rsum"][:, None]


def _logprobs_grad(st, case):
    T, tokens = case["temperature"], st["tokens"].long()
    live = (tokens >= 0).float()      # (the gradients of a row that is left out are zero)
    dlogp, dent = st["d_logp"] * live, st["d_entropy"] * live
    y, p = _given(st, T)
    lp = y.sub_(st["rsum"].log()[:, None])
    g = p * (-dlogp[:, None] - dent[:, None] * (lp + st["entropy"][:, None]))
    g.scatter_add_(1, tokens.clamp(min=0)[:, None], dlogp[:, None])
    return g.div_(T).to(DT[case["d"]])


def _teacher(st, T):
    """q, ln q (0 where there is no entry) and whether the row has any."""
    has = st["ids"] >= 0
    live = has.any(1)
    t = st["teacher"].masked_fill(~has, -math.inf) / T
    t = t - torch.where(live, t.amax(1), torch.zeros_like(t[:, 0]))[:, None]
    e = t.exp()
    s = e.sum(1, keepdim=True).clamp(min=1e-30)
    return e / s, torch.where(has, t - s.log(), torch.zeros_like(t)), live


def _distill_dx(st, case, p, q, live):
    w = torch.where(live, st["weight"], torch.zeros_like(st["weight"])) / case["temperature"]
    g = p.mul_(w[:, None])
    g.scatter_add_(1, st["ids"].clamp(min=0).long(), -q * w[:, None])
    return g.to(DT[case["d"]])


def _distill(st, case):
    T = case["temperature"]
    q, lq, live = _teacher(st, T)
    y, m, e, s = _stats(st, T)
    zero = torch.zeros(st["n"], device="cuda")
    at = y.gather(1, st["ids"].clamp(min=0).long()) - s.log()
    loss = torch.where(live, (q * (lq - at)).sum(1), zero)
    res = (loss, torch.where(live, m[:, 0], zero), torch.where(live, s[:, 0], zero))
    if not case["d"]:
        return res
    del y
    return res + (_distill_dx(st, case, e.div_(s), q, live),)


def _distill_grad(st, case):
    q, _, live = _teacher(st, case["temperature"])
    y, p = _given(st, case["temperature"])
    del y
    return _distill_dx(st, case, p, q, live)


# --------------------------------------------------------------------------
# the definitions in 64 bits
# --------------------------------------------------------------------------
def exact(case, seed):
    st = prepare(case, seed)
    n, V, T, op = case["rows"], case["vocab"], case["temperature"], case["op"]
    outs = []
    # (64-bit values of whole gradients, in bytes: left to the plain form beyond what fits beside them)
    if case.get("d") and n * V > 1 << 30:
        return None
    for b in _blocks(n, V):
        x = st["x"][b].double()
        rows = range(b.start, b.stop)
        logz = torch.logsumexp(x / T, 1)
        big = x.amax(1)
        if op.startswith("logprobs"):
            tok = st["tokens"][b].long()
            live = tok >= 0
            at = tok.clamp(min=0)[:, None]
        else:
            live = (st["ids"][b] >= 0).any(1)
            q = torch.zeros(len(rows), V, dtype=torch.float64, device="cuda")
            t = st["teacher"][b].double().masked_fill(st["ids"][b] < 0, -math.inf) / T
            qk = torch.where(live[:, None], torch.softmax(t, 1), torch.zeros_like(t)).nan_to_num(0.0)
        if op == "logprobs":
            lp = x / T - logz[:, None]
            p = torch.softmax(x / T, 1)
            ent = -torch.xlogy(p, p).sum(1)
            res = [lp.gather(1, at)[:, 0], ent, big, torch.exp(logz - big / T)]
            res = [torch.where(live, r, torch.zeros_like(r)) for r in res]
            if case["k"]:
                best = lp.topk(min(case["k"], V), dim=1).values      # (the values do not depend on the order of ties)
                res += [None, torch.where(live[:, None], best, torch.zeros_like(best))]
        elif op == "distill":
            lp = torch.gather(x, 1, st["ids"][b].clamp(min=0).long()) / T - logz[:, None]
            terms = torch.where(qk > 0, torch.xlogy(qk, qk) - qk * lp, torch.zeros_like(qk))
            res = [torch.where(live, r, torch.zeros_like(r)) for r in (terms.sum(1), big, torch.exp(logz - big / T))]
            if case["d"]:
                q.scatter_add_(1, st["ids"][b].clamp(min=0).long(), qk)
                w = torch.where(live, st["weight"][b].double(), torch.zeros_like(big)) / T
                res.append((torch.softmax(x / T, 1) - q) * w[:, None])
        else:
            # from what the forward pass left
            p = torch.exp((x - st["rmax"][b].double()[:, None]) / T) / st["rsum"][b].double()[:, None]
            if op == "distill_grad":
                q.scatter_add_(1, st["ids"][b].clamp(min=0).long(), qk)
                w = torch.where(live, st["weight"][b].double(), torch.zeros_like(big)) / T
                res = [(p - q) * w[:, None]]
            else:
                hot = torch.zeros_like(x).scatter_(1, at, 1.0)
                d = hot.sub_(p).mul_(st["d_logp"][b].double()[:, None])
                d -= st["d_entropy"][b].double()[:, None] * (torch.xlogy(p, p) + p * st["entropy"][b].double()[:, None])
                res = [torch.where(live[:, None], d / T, torch.zeros_like(d))]
        outs.append(res)
    whole = [None if col[0] is None else torch.cat(col) for col in zip(*outs)]
    return whole[0] if len(whole) == 1 else tuple(whole)
