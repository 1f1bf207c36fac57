"""Plain 64-bit restatements of the 4-bit cache, the attention over it and the
verification of drafted tokens (numpy), and seeded inputs for their tests."""
from __future__ import annotations

import numpy as np

FIELD = [(e >> 1) + 4 * (e & 1) for e in range(8)]      # which 4-bit field of a word holds value e


def round_bits(x, bits):
    """x rounded to `bits` significant bits, ties to even (float64 in and out)."""
    m, e = np.frexp(x)
    return np.ldexp(np.round(np.ldexp(m, bits)), e - bits)


def quantize(x):
    """x float32 [..., dim] -> n int8 [..., dim], d float16 [..., dim / 32]: tk_kv_append's rule, in fp32 steps."""
    x = np.asarray(x, np.float32)
    b = np.where(np.isfinite(x), x, np.float32(0)).reshape(*x.shape[:-1], -1, 32)
    first = np.abs(b).argmax(-1)                         # numpy's argmax: the first of several
    m = np.take_along_axis(b, first[..., None], -1)[..., 0]
    d = np.clip(round_bits((m * np.float32(-0.125)).astype(np.float64), 8), -8160, 8160).astype(np.float16) + np.float16(0)
    d32 = d.astype(np.float32)
    with np.errstate(divide="ignore"):
        r = np.where(d32 == 0, np.float32(0), np.float32(1) / d32).astype(np.float32)
    t = (b * r[..., None]).astype(np.float32) + np.float32(8.5)
    n = np.clip(np.floor(t), 0, 15).astype(np.int8) - 8
    return n.reshape(x.shape), d


def pack(n):
    """n int8 [..., dim] -> bytes [..., dim / 2]."""
    w = np.zeros((*n.shape[:-1], n.shape[-1] // 8), np.uint32)
    g = (n.reshape(*w.shape, 8).astype(np.int32) & 15).astype(np.uint32)
    for e in range(8):
        w |= g[..., e] << np.uint32(4 * FIELD[e])
    return w.view(np.uint8)


def unpack(q, s):
    """Bytes and scales -> values, float64."""
    w = np.ascontiguousarray(q).view(np.uint32)
    n = np.stack([((w >> np.uint32(4 * FIELD[e])) & 15).astype(np.int64) for e in range(8)], -1)
    n = np.where(n > 7, n - 16, n).reshape(*w.shape[:-1], -1)
    with np.errstate(invalid="ignore"):               # infinite scales of rows that nothing reads
        return n * np.repeat(s.astype(np.float64), 32, -1)


def random_cache(rng, n_pages, page, heads, dim, garbage=False):
    """Cache planes with every whole number and both signs of scale; `garbage`: NaN and infinite scales."""
    q = [rng.integers(0, 256, (n_pages, heads, page, dim // 2), dtype=np.uint8) for _ in "kv"]
    s = []
    for _ in "kv":
        d = round_bits(rng.standard_normal((n_pages, heads, page, dim // 32)) * 0.12, 8).astype(np.float16)
        if garbage:
            d[...] = rng.choice(np.array([np.nan, np.inf, -np.inf, 65504.0], np.float16), d.shape)
        s.append(d)
    return {"k_q": q[0], "k_s": s[0], "v_q": q[1], "v_s": s[1]}


def batch(rng, new, kv, page, spare=3):
    """q_start, kv_len, pages (a random placement; unused entries name page 0) and the number of pages."""
    need = [-(-c // page) for c in kv]
    total, width = sum(need) + spare, max(1, max(need))
    order = rng.permutation(total).astype(np.int32)
    pages, at = np.zeros((len(kv), width), np.int32), 0
    for b, n in enumerate(need):
        pages[b, :n] = order[at:at + n]
        at += n
    return np.concatenate([[0], np.cumsum(new)]).astype(np.int32), np.array(kv, np.int32), pages, total


def attend(cache, q_start, kv_len, pages, q, heads, kv_heads, dim, scale, window):
    """(out, reach) float64 [tokens, heads, dim]; reach = sum_j p_j |v_j|, what rounding errors are relative to."""
    q = np.asarray(q, np.float64).reshape(-1, heads, dim)
    out, reach = np.zeros_like(q), np.zeros_like(q)
    page = cache["k_q"].shape[2]
    for b in range(len(kv_len)):
        r0, r1, c = int(q_start[b]), int(q_start[b + 1]), int(kv_len[b])
        if r1 == r0 or c == 0:
            continue
        ids = pages[b, : -(-c // page)]
        k, v = (unpack(cache[x + "_q"][ids], cache[x + "_s"][ids]).transpose(1, 0, 2, 3).reshape(kv_heads, -1, dim)[:, :c]
                for x in "kv")
        for i in range(r1 - r0):
            pos = c - (r1 - r0) + i
            lo = max(0, pos - window + 1) if window else 0
            if pos < 0:
                continue
            for h in range(heads):
                g = h // (heads // kv_heads)
                s = scale * (k[g, lo:pos + 1] @ q[r0 + i, h])
                p = np.exp(s - s.max())
                p /= p.sum()
                out[r0 + i, h] = p @ v[g, lo:pos + 1]
                reach[r0 + i, h] = p @ np.abs(v[g, lo:pos + 1])
    return out, reach


def verify(target, tokens, row_start, u_accept, u_sample, draft, temperature):
    """n_accept, next, logp by the definition, with the weights of tk_draft_verify: powers of two relative to the
    row's largest whole exponent, the sum in 64 bits rounded once to fp32, draws in whole multiples of 2^-38."""
    f32 = np.float32
    c = f32(1.4426950408889634 / (temperature or 1.0))

    def row(x):
        y = (x.astype(f32) * c).astype(f32)
        i = np.floor(y)
        top = i.max()
        with np.errstate(invalid="ignore"):
            w = np.where(i - top >= -100, np.exp2((y - i).astype(np.float64)).astype(f32) * np.exp2(i - top).astype(f32), f32(0))
        return np.nan_to_num(w).astype(f32), f32(w.astype(np.float64).sum())

    n_acc, nxt, logp = [], [], np.zeros(len(target))
    for b in range(len(row_start) - 1):
        r0, r1 = int(row_start[b]), int(row_start[b + 1])
        for r in range(r0, r1):
            last = r == r1 - 1
            lp = target[r].astype(np.float64) / (temperature or 1.0)
            lp = lp - lp.max()
            lp = lp - np.log(np.exp(lp).sum())
            x = -1 if last else int(tokens[r + 1])
            known = 0 <= x < target.shape[1]
            if temperature == 0:
                tok = int(target[r].argmax())
                ok = not last and x == tok
            else:
                w, s = row(target[r])
                p = (w / s).astype(f32)
                q = np.zeros_like(p)
                if not last and draft is not None:
                    w2, s2 = row(draft[r])
                    q = (w2 / s2).astype(f32)
                elif known:
                    q[x] = 1
                ok = known and f32(u_accept[r]) * q[x] < p[x]
                if not ok:
                    left = (np.maximum(p - q, 0) * f32(2.0 ** 38)).astype(np.int64) if not last else \
                        (p * f32(2.0 ** 38)).astype(np.int64)
                    if left.sum() == 0:
                        left = (p * f32(2.0 ** 38)).astype(np.int64)
                    goal = int(left.sum()) * int(f32(u_sample[b]) * f32(2 ** 24)) >> 24
                    tok = int((left.cumsum() > goal).argmax())
            if ok:
                logp[r] = lp[x]
                continue
            logp[r] = lp[tok]
            n_acc.append(r - r0)
            nxt.append(tok)
            break
    return np.array(n_acc, np.int32), np.array(nxt, np.int32), logp
