"""Measured cases of the serving operators: the 4-bit key/value cache (append
and read back), attention over it, and the verification of drafted tokens.

Shapes: the attention cases are the decoder layer of the framework's own
configurations (32 query heads x 128, 8 key/value heads x 128) and smaller
generic ones; the vocabulary is its LM head's (262144) and generic ones.

The cache (one layer): k_q, v_q uint8 [pages, kv_heads, page, dim/2] and k_s,
v_s float16 [pages, kv_heads, page, dim/32].  32 consecutive values share one
scale d, of 8 significant bits, and are held as whole numbers n in -8..7,
value n*d (exact in float16).  A 32-bit word of k_q/v_q holds 8 consecutive
values: value e in bits 4*((e >> 1) + 4*(e & 1)) .. +3, two's complement.
A sequence's token t lives in page pages[seq, t // page], row t % page.

The new tokens of a call are packed: sequence b has tokens
q_start[b] .. q_start[b+1]-1, the last ones of its kv_len[b] cached tokens.
"""
import math
import random

import torch

own = False

DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
LOG2E = math.log2(math.e)


# --------------------------------------------------------------------------
# cases
# --------------------------------------------------------------------------
def listed():
    layer = dict(heads=32, kv_heads=8, dim=128, page=64)
    return [
        # one decode step of 16 users: the engine's fp32 rows go into the cache (launch latency)
        dict(name="append_decode_16", op="append", kv_heads=8, dim=128, page=64, dtype="f32", seqs=16, new=1, kv=2049,
             ragged=True, shape=1),
        # a packed batch of prompts, odd lengths, behind what is cached already (bandwidth)
        dict(name="append_prompts", op="append", kv_heads=8, dim=128, page=64, dtype="bf16", seqs=5, new=4093, kv=5000,
             ragged=True, shape=2),
        # one user, one token, a chat's context (latency)
        dict(name="decode_1", op="attend", dtype="f16", seqs=1, new=1, kv=4097, ragged=False, window=0, shape=3, **layer),
        # a serving batch of single tokens with contexts of very different length
        dict(name="decode_32_ragged", op="attend", dtype="bf16", seqs=32, new=1, kv=16300, ragged=True, window=0, shape=4,
             **layer),
        # one token against a long document
        dict(name="decode_long", op="attend", dtype="f32", seqs=1, new=1, kv=131071, ragged=False, window=0, shape=5, **layer),
        # five rows per user: a pending token and four drafted ones, the engine's fp32
        dict(name="drafted_8x5", op="attend", dtype="f32", seqs=8, new=5, kv=8191, ragged=False, window=0, shape=6, **layer),
        # a whole prompt from nothing: the compute-bound end
        dict(name="prompt_8192", op="attend", dtype="bf16", seqs=1, new=8192, kv=8192, ragged=False, window=0, shape=7,
             **layer),
        # chunks of prompts behind cached context, 64-wide heads, small pages, a sliding window
        dict(name="chunks_window", op="attend", dtype="f16", seqs=3, new=1000, kv=6001, ragged=True, window=1024, shape=8,
             heads=16, kv_heads=4, dim=64, page=16),
        # an engine prompt in fp32, held to fp32 accuracy
        dict(name="prompt_f32", op="attend", dtype="f32", seqs=2, new=1537, kv=2000, ragged=True, window=0, shape=9, **layer),
        # one user, four tokens drafted by lookup (no draft distribution), the LM head's vocabulary
        dict(name="verify_1x4", op="verify", seqs=1, new=5, vocab=262144, draft=False, temperature=1.0, ragged=False, shape=10),
        # a batch with a draft model's distributions, up to seven drafts each
        dict(name="verify_24x7", op="verify", seqs=24, new=8, vocab=262144, draft=True, temperature=0.8, ragged=True, shape=11),
        # greedy verification with an odd vocabulary
        dict(name="verify_greedy", op="verify", seqs=64, new=5, vocab=50257, draft=False, temperature=0.0, ragged=True,
             shape=12),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("append", "attend", "attend", "attend", "verify"))
    shape = rng.randrange(1 << 20)
    if op == "verify":
        vocab, new = _log(rng, 1000, 262144), rng.randint(1, 8)
        seqs = max(1, min(_log(rng, 1, 64), 24 * 8 * 262144 // (vocab * new)))
        return dict(op=op, seqs=seqs, new=new, vocab=vocab, draft=rng.random() < 0.5,
                    temperature=rng.choice((0.0, 0.6, 1.0, 1.3)), ragged=rng.random() < 0.5, shape=shape)
    heads, kv_heads = rng.choice(((32, 8), (32, 4), (16, 4), (16, 8), (8, 8), (8, 1)))
    dim, page = rng.choice((64, 128)), rng.choice((16, 32, 64, 128))
    dtype, ragged = rng.choice(("f32", "f16", "bf16")), rng.random() < 0.6
    if op == "append":
        seqs = _log(rng, 1, 32)
        new = _log(rng, 1, 8192 // seqs)
        return dict(op=op, kv_heads=kv_heads, dim=dim, page=page, dtype=dtype, seqs=seqs, new=new,
                    kv=new + _log(rng, 1, 8192), ragged=ragged, shape=shape)
    if rng.random() < 0.6:                      # tokens being generated
        seqs, new = _log(rng, 1, 32), rng.choice((1, 1, 1, rng.randint(2, 8)))
        kv = max(new, _log(rng, 1, 131072 // seqs))
    else:                                       # prompts, whole or in chunks
        seqs = _log(rng, 1, 8)
        new = _log(rng, 9, 4096 // seqs)
        kv = new + rng.choice((0, _log(rng, 1, 4096)))
    return dict(op=op, heads=heads, kv_heads=kv_heads, dim=dim, page=page, dtype=dtype, seqs=seqs, new=new, kv=kv,
                ragged=ragged, window=rng.choice((0, 0, 0, _log(rng, 1, 4096))), shape=shape)


def lens(case):
    """New tokens and cached tokens of each sequence: the case's own, whatever the seed of its values."""
    r = random.Random(case["shape"])
    new, kv = [], []
    for b in range(case["seqs"]):
        full = not case["ragged"] or b == 0
        n = case["new"] if full else r.randint(1, case["new"])
        new.append(n)
        if "kv" in case:
            kv.append(case["kv"] if full else max(n, _log(r, max(1, case["kv"] // 16), case["kv"])))
    return new, kv


def work(case):
    new, kv = lens(case)
    n = sum(new)
    if case["op"] == "verify":
        drafted = (n - len(new)) if case["draft"] else 0
        return {"bytes": 4.0 * case["vocab"] * (n + drafted) + 16 * n, "flops": 4.0 * case["vocab"] * (n + drafted)}
    held = case["kv_heads"] * 2 * (case["dim"] // 2 + case["dim"] // 16)      # bytes of one cached token
    size = 4 if case["dtype"] == "f32" else 2
    if case["op"] == "append":
        values = n * case["kv_heads"] * case["dim"] * 2
        return {"bytes": float(values * size + n * held + values * 2), "flops": 4.0 * values}
    w = case["window"]
    pairs = read = 0
    for a, c in zip(new, kv):
        first = max(0, c - a - w + 1) if w else 0          # the first key that any row sees
        read += c - first
        if not w:
            pairs += a * (c - a) + a * (a + 1) // 2
        else:
            pairs += sum(min(w, c - a + i + 1) for i in range(a))
    return {"bytes": float(2 * n * case["heads"] * case["dim"] * size + read * held),
            "flops": 4.0 * pairs * case["heads"] * case["dim"]}


# --------------------------------------------------------------------------
# the cache's numbers in elementary operations
# --------------------------------------------------------------------------
def quantize(x):
    """x [..., dim] float32 -> whole numbers n [..., dim] (int32, -8..7) and scales d [..., dim/32] (float32).
    d = m / -8, m the value of largest magnitude (the first of several), in 8 significant bits and in
    float16's range; n = floor(x / d + 1/2), clamped."""
    b = x.unflatten(-1, (-1, 32))
    m = b.gather(-1, b.abs().max(-1, keepdim=True).values.eq(b.abs()).to(torch.uint8).argmax(-1, keepdim=True))
    d = (m * -0.125).to(torch.bfloat16).float().clamp(-8160.0, 8160.0).to(torch.float16).float()
    r = torch.where(d == 0, torch.zeros_like(d), 1.0 / d)
    n = (b * r + 8.5).floor().clamp(0, 15) - 8
    return n.to(torch.int32).flatten(-2), d.squeeze(-1)


_SHIFT = [4 * ((e >> 1) + 4 * (e & 1)) for e in range(8)]


def pack(n):
    """Whole numbers [..., dim] -> the cache's bytes [..., dim/2]."""
    w = (n.unflatten(-1, (-1, 8)).to(torch.int64) & 15) << torch.tensor(_SHIFT, device=n.device)
    w = w.sum(-1)
    return torch.where(w >= 1 << 31, w - (1 << 32), w).to(torch.int32).view(torch.uint8)


def unpack(q, s):
    """The cache's bytes [..., dim/2] and scales [..., dim/32] -> values [..., dim], float32."""
    w = q.contiguous().view(torch.int32).unsqueeze(-1) >> torch.tensor(_SHIFT, dtype=torch.int32, device=q.device)
    n = (((w & 15) ^ 8) - 8).flatten(-2).float()
    return (n.unflatten(-1, (-1, 32)) * s.float().unsqueeze(-1)).flatten(-2)


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


def _normal(g, *size, dtype=torch.float32):
    return torch.randn(*size, generator=g, device="cuda").to(dtype)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    new, kv = lens(case)
    start = [0]
    for n in new:
        start.append(start[-1] + n)
    n, B = start[-1], len(new)
    st = {"case": case, "n": n, "max_new": max(new), "q_start": torch.tensor(start, dtype=torch.int32, device="cuda")}
    if case["op"] == "verify":
        # a trained model's rows: a few likely tokens above a wide tail; the draft model is near the target
        V = case["vocab"]
        t = _normal(g, n, V) * 2.0
        top = torch.randint(V, (n, 32), generator=g, device="cuda")
        t.scatter_add_(1, top, 6.0 + 4.0 * torch.rand(n, 32, generator=g, device="cuda"))
        d = t + 0.7 * _normal(g, n, V)
        temp = case["temperature"] or 1.0
        if case["draft"]:   # drawn from the draft's distribution; a lookup's draft is mostly the likeliest token
            drafted = (d / temp - torch.log(-torch.log(torch.rand(n, V, generator=g, device="cuda")))).argmax(1)
        else:
            drafted = torch.where(torch.rand(n, generator=g, device="cuda") < 0.8, t.argmax(1), top[:, 0])
        tokens = torch.zeros(n, dtype=torch.int32, device="cuda")
        tokens[1:] = drafted[:-1].to(torch.int32)          # row i judges the token at row i + 1
        st |= {"target": t, "draft": d if case["draft"] else None, "tokens": tokens,
               "u_accept": torch.rand(n, generator=g, device="cuda"), "u_sample": torch.rand(B, generator=g, device="cuda"),
               "accepted": torch.zeros(B, dtype=torch.int32, device="cuda"),
               "next": torch.zeros(B, dtype=torch.int32, device="cuda"), "logp": torch.zeros(n, device="cuda")}
        return st
    P, H, D, dtype = case["page"], case["kv_heads"], case["dim"], DT[case["dtype"]]
    need = [-(-c // P) for c in kv]
    width, total = max(need), sum(need)
    order = torch.randperm(total, generator=g, device="cuda").to(torch.int32)
    at = torch.tensor([sum(need[:b]) for b in range(B)], dtype=torch.int64, device="cuda")
    col = torch.arange(width, device="cuda")
    has = col[None] < torch.tensor(need, device="cuda")[:, None]
    st["pages"] = torch.where(has, order[(at[:, None] + col[None]).clamp(max=total - 1)], torch.zeros((), dtype=torch.int32,
                                                                                                     device="cuda")).contiguous()
    st["kv_len"] = torch.tensor(kv, dtype=torch.int32, device="cuda")
    # keys have a few channels that stand out, as trained models' do; values do not
    loud = 1.0 + 3.0 * (torch.rand(H, 1, D, generator=g, device="cuda") > 0.97)
    if case["op"] == "append":
        for x in ("k", "v"):
            st[x + "_q"] = torch.zeros(total, H, P, D // 2, dtype=torch.uint8, device="cuda")
            st[x + "_s"] = torch.zeros(total, H, P, D // 32, dtype=torch.float16, device="cuda")
            st[x + "_out"] = torch.zeros(n, H * D, dtype=torch.float16, device="cuda")
        st["k"] = (_normal(g, n, H, D) * loud[:, 0]).flatten(1).to(dtype)
        st["v"] = _normal(g, n, H * D, dtype=dtype)
    else:
        for x, f in (("k", loud), ("v", 1.0)):
            q, s = [], []
            for some in torch.arange(total).split(4096):
                m, d = quantize(_normal(g, len(some), H, P, D) * f)
                q.append(pack(m))
                s.append(d.to(torch.float16))
            st[x + "_q"], st[x + "_s"] = torch.cat(q), torch.cat(s)
        st["q"] = _normal(g, n, case["heads"] * D, dtype=dtype)
        st["out"] = torch.zeros(n, case["heads"] * D, dtype=dtype, device="cuda")
    if own:   # the descriptors of the cache and of the batch, which a program makes once
        tk, _ = _framework()
        st["cache"] = tk.make_kvcache(st["k_q"], st["k_s"], st["v_q"], st["v_s"])
        st["seqs"] = tk.make_seqs(st["q_start"], st["kv_len"], st["pages"], n, st["max_new"])
    return st


# --------------------------------------------------------------------------
# one pass
# --------------------------------------------------------------------------
def run(st):
    case = st["case"]
    if own:
        return _run_own(st, case)
    return {"append": _append, "attend": _attend, "verify": _verify}[case["op"]](st, case)


def _run_own(st, case):
    tk, ctx = _framework()
    if case["op"] == "verify":
        ctx.draft_verify(st["target"], st["tokens"], st["q_start"], st["u_accept"], st["u_sample"], st["accepted"], st["next"],
                         st["logp"], draft=st["draft"], temperature=case["temperature"])
        return st["accepted"], st["next"], st["logp"]
    dt = {"f32": tk.DT_F32, "f16": tk.DT_F16, "bf16": tk.DT_BF16}[case["dtype"]]
    if case["op"] == "append":
        ctx.kv_append(st["cache"], st["seqs"], st["k"], st["v"], x_dtype=dt)
        ctx.kv_read(st["cache"], st["seqs"], st["k_out"], st["v_out"], out_dtype=tk.DT_F16)
        return st["k_out"], st["v_out"]
    ctx.kv_attend(st["cache"], st["seqs"], st["q"], case["heads"], st["out"], x_dtype=dt, window=case["window"])
    return st["out"]


def _where(st):
    """Sequence and position of each new token."""
    i = torch.arange(st["n"], device="cuda", dtype=torch.int32)
    seq = torch.searchsorted(st["q_start"], i, right=True) - 1
    return seq, st["kv_len"][seq] - (st["q_start"][seq + 1] - i)


def _append(st, case):
    seq, pos = _where(st)
    P = case["page"]
    page, row = st["pages"][seq, pos // P].long(), (pos % P).long()
    got = []
    for x in ("k", "v"):
        m, d = quantize(st[x].float().unflatten(-1, (case["kv_heads"], case["dim"])))
        q, s = pack(m), d.to(torch.float16)
        st[x + "_q"][page, :, row] = q
        st[x + "_s"][page, :, row] = s
        got.append(unpack(q, s).flatten(1).to(torch.float16))
    return tuple(got)


def _attend(st, case):
    H, Hk, D = case["heads"], case["kv_heads"], case["dim"]
    seq, pos = _where(st)
    pages = st["pages"].long()
    B, L = pages.shape[0], pages.shape[1] * case["page"]
    k, v = (unpack(st[x + "_q"], st[x + "_s"])[pages].transpose(1, 2).reshape(B, Hk, L, D) for x in ("k", "v"))
    at = torch.arange(st["n"], device="cuda") - st["q_start"][seq]
    q = torch.zeros(B, st["max_new"], H, D, device="cuda")
    q[seq, at] = st["q"].float().view(-1, H, D)
    where = torch.full((B, st["max_new"]), -1, dtype=torch.int64, device="cuda")
    where[seq, at] = pos.long()
    q = q.view(B, -1, Hk, H // Hk, D).permute(0, 2, 3, 1, 4).reshape(B, Hk, -1, D)
    s = torch.matmul(q, k.transpose(-1, -2)).mul_(1.0 / math.sqrt(D)).view(B, Hk, H // Hk, -1, L)
    key = torch.arange(L, device="cuda")
    seen = key <= where[..., None]
    if case["window"]:
        seen &= key > where[..., None] - case["window"]
    s.masked_fill_(~seen[:, None, None], -math.inf)
    m = s.amax(-1, keepdim=True)
    p = s.sub_(torch.where(m == -math.inf, torch.zeros_like(m), m)).exp_()
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p.view(B, Hk, -1, L), v).view(B, Hk, H // Hk, -1, D) / torch.where(total == 0, torch.ones_like(total), total)
    return o.permute(0, 3, 1, 2, 4).reshape(B, -1, H * D)[seq, at].to(DT[case["dtype"]])


def _weights(x, c):
    """2^(c x) of each row, with the largest in [1, 2): values, and the row's sum (64 bits) as float32."""
    y = x * c
    i = y.floor()
    top = i.amax(1, keepdim=True)
    e = torch.exp2(y - i) * torch.exp2((i - top).clamp(min=-100.0))
    e = torch.where(i - top < -100.0, torch.zeros_like(e), e)
    return e, e.sum(1, dtype=torch.float64).to(torch.float32), top.squeeze(1), y


def _verify(st, case):
    t, d, T = st["target"], st["draft"], case["temperature"]
    n, B = st["n"], case["seqs"]
    c = torch.tensor(LOG2E / (T or 1.0), dtype=torch.float32, device="cuda")
    row = torch.arange(n, device="cuda")
    seq, last = torch.searchsorted(st["q_start"].long(), row, right=True) - 1, st["q_start"].long()[1:] - 1
    judged = torch.cat([st["tokens"][1:], st["tokens"][:1]]).long()          # the token that row i judges
    e, S, top, y = _weights(t, c)
    if T:
        p = (e / S[:, None]).gather(1, judged[:, None]).squeeze(1)
        if d is not None:
            f, Sd, _, _ = _weights(d, c)
            q = (f / Sd[:, None]).gather(1, judged[:, None]).squeeze(1)
        else:
            q = torch.ones_like(p)
        ok = st["u_accept"] * q < p
    else:
        best = t.argmax(1)
        ok = judged == best
    ok &= row != last[seq]
    stop = torch.full((B,), n, dtype=torch.int64, device="cuda").scatter_reduce(0, seq, torch.where(ok, n, row), "amin")
    accepted = stop - st["q_start"].long()[:-1]
    if T:
        w = e[stop] / S[stop, None]
        r = torch.zeros_like(w)
        if d is not None:
            r = torch.where((stop != last)[:, None], f[stop] / Sd[stop, None], r)
        else:
            r.scatter_(1, judged[stop, None], torch.where(stop != last, 1.0, 0.0)[:, None])
        left = ((w - r).clamp(min=0) * 2.0 ** 38).to(torch.int64)
        left = torch.where(left.sum(1, keepdim=True) == 0, (w * 2.0 ** 38).to(torch.int64), left)
        upto = left.cumsum(1)
        goal = (upto[:, -1] * (st["u_sample"] * 2.0 ** 24).to(torch.int64)) >> 24
        token = (upto > goal[:, None]).to(torch.uint8).argmax(1)
    else:
        token = best[stop]
    said = judged.scatter(0, stop, token)
    logp = ((y.gather(1, said[:, None]).squeeze(1) - top) - torch.log2(S)) * math.log(2.0)
    logp = torch.where(row <= stop[seq], logp, torch.zeros_like(logp))
    return accepted.to(torch.int32), token.to(torch.int32), logp


# --------------------------------------------------------------------------
# the definitions in 64 bits
# --------------------------------------------------------------------------
def exact(case, seed):
    st = prepare(case, seed)
    new, kv = lens(case)
    first = [sum(new[:b]) for b in range(len(new))]
    if case["op"] == "append":
        res = []
        for x in ("k", "v"):
            b = st[x].double().view(st["n"], -1, 32)
            big, where = b.abs().max(-1)
            sign = torch.sign(b.gather(-1, (b.abs() == big[..., None]).int().argmax(-1, keepdim=True)))[..., 0]
            # 8 significant bits, to nearest even, on float16's grid
            d = big / 8
            unit = torch.exp2(torch.floor(torch.log2(d.clamp(min=1e-300))) - 7)
            d = -sign * (torch.round(d / unit) * unit).clamp(max=8160.0).to(torch.float16).double()
            n = torch.floor(b / torch.where(d == 0, torch.ones_like(d), d)[..., None] + 0.5).clamp(-8, 7)
            res.append((n * d[..., None]).reshape(st["n"], -1))
        return tuple(res)
    if case["op"] == "attend":
        H, Hk, D, P = case["heads"], case["kv_heads"], case["dim"], case["page"]
        out = torch.zeros(st["n"], H, D, dtype=torch.float64, device="cuda")
        for b, (a, c) in enumerate(zip(new, kv)):
            pages = st["pages"][b, : -(-c // P)].long()
            held = []
            for x in ("k", "v"):
                raw, s = st[x + "_q"][pages].long(), st[x + "_s"][pages].double()
                vals = torch.zeros(*raw.shape[:-1], D, dtype=torch.float64, device="cuda")
                for e in range(8):      # value e of each group of 8: the low or high half of one of its 4 bytes
                    field = (e >> 1) + 4 * (e & 1)
                    nib = (raw[..., field // 2 :: 4] >> (4 * (field % 2))) & 15
                    vals[..., e::8] = torch.where(nib > 7, nib - 16, nib).double()
                vals *= s.repeat_interleave(32, dim=-1)
                held.append(vals.permute(1, 0, 2, 3).reshape(Hk, -1, D)[:, :c])
            key = torch.arange(c, device="cuda")
            for lo in range(0, a, 1024):
                q = st["q"][first[b] + lo : first[b] + min(a, lo + 1024)].double().view(-1, Hk, H // Hk, D)
                pos = c - a + lo + torch.arange(q.shape[0], device="cuda")
                hide = (key[None] > pos[:, None]) | ((key[None] <= pos[:, None] - case["window"]) if case["window"] else False)
                s = torch.einsum("nhgd,hkd->nhgk", q, held[0]) / math.sqrt(D)
                s.masked_fill_(hide[:, None, None], -math.inf)
                out[first[b] + lo : first[b] + lo + q.shape[0]] = torch.einsum("nhgk,hkd->nhgd", torch.softmax(s, -1),
                                                                               held[1]).reshape(-1, H, D)
        return out.flatten(1)
    # the decisions from probabilities in 64 bits; as whole numbers they have no 64-bit value, their log-probabilities do
    logp = torch.zeros(st["n"], dtype=torch.float64, device="cuda")
    T = case["temperature"]
    for b, a in enumerate(new):
        for r in range(first[b], first[b] + a):
            lp = torch.log_softmax(st["target"][r].double() / (T or 1.0), 0)
            p, q = lp.exp(), torch.zeros_like(lp)
            bonus = r == first[b] + a - 1
            x = 0 if bonus else int(st["tokens"][r + 1])
            if not bonus:
                if st["draft"] is not None:
                    q = torch.softmax(st["draft"][r].double() / (T or 1.0), 0)
                else:
                    q[x] = 1.0
            best = int(lp.argmax())
            if not bonus and (float(st["u_accept"][r]) * float(q[x]) < float(p[x]) if T else x == best):
                logp[r] = lp[x]
                continue
            upto = (p - q).clamp(min=0).cumsum(0)
            token = int((upto > float(st["u_sample"][b]) * upto[-1]).int().argmax()) if T else best
            logp[r] = lp[token]
            break
    return None, None, logp
