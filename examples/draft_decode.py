"""Drafted decoding with a small random decoder: block-quantized projections
(Q4_K, the decode GEMV), a 4-bit key/value cache, attention over it, an fp16 LM
head and the verification of drafted tokens.

Each step runs every sequence's pending token and its drafts through the model
at once (a few rows per sequence, the decode GEMV reads each weight once), adds
their keys and values to the cache, and keeps what tk_draft_verify accepts.
Rejected tokens stay in the cache behind the sequence's length and are
overwritten by the next step.  Drafts are looked up: what followed the last
occurrence of the last token in the sequence's own text.

usage: python examples/draft_decode.py [--steps N] [--drafts K] [--temperature T] [--seqs B]
"""
from __future__ import annotations

import argparse
import sys
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parents[1]))
import tier_b200 as tk  # noqa: E402

MAX_ROWS = 16          # tk_gemv takes 1..16 tokens


class Decoder:
    """A random decoder whose weights live on the device as the engine keeps them."""

    def __init__(self, ctx, layers=2, hidden=512, heads=8, kv_heads=2, head_dim=64, ffn=1024, vocab=1000, seqs=3,
                 max_tokens=512, page_tokens=32, seed=0):
        self.ctx, self.vocab, self.hidden = ctx, vocab, hidden
        self.heads, self.kv_heads, self.head_dim, self.ffn = heads, kv_heads, head_dim, ffn
        g = torch.Generator(device="cuda").manual_seed(seed)

        def matrix(rows, cols):
            w = torch.randn(rows, cols, generator=g, device="cuda") * cols ** -0.5
            blocks = torch.empty(rows, tk.row_bytes(tk.Q4_K, cols), dtype=torch.uint8, device="cuda")
            return ctx.quantize(tk.Q4_K, w, rows, cols, blocks)

        q, kv = heads * head_dim, kv_heads * head_dim
        self.layers = [{"q": matrix(q, hidden), "k": matrix(kv, hidden), "v": matrix(kv, hidden), "o": matrix(hidden, q),
                        "gate": matrix(ffn, hidden), "up": matrix(ffn, hidden), "down": matrix(hidden, ffn)}
                       for _ in range(layers)]
        self.embed = torch.randn(vocab, hidden, generator=g, device="cuda")
        self.head = (torch.randn(vocab, hidden, generator=g, device="cuda") * 3 * hidden ** -0.5).half()
        # one cache per layer; sequence b owns pages b * per .. b * per + per - 1
        per = -(-max_tokens // page_tokens)
        self.caches = [tk.alloc_kvcache(seqs * per, page_tokens, kv_heads, head_dim) for _ in range(layers)]
        self.pages = torch.arange(seqs * per, dtype=torch.int32, device="cuda").view(seqs, per)

    def _gemv(self, names, weights, x, sizes):
        n = x.shape[0]
        ys = [torch.empty(n, s, device="cuda") for s in sizes]
        if len(names) == 1:
            self.ctx.gemv(tk.Q4_K, weights[names[0]], sizes[0], x.shape[1], x, ys[0], M=n)
        else:
            self.ctx.gemv_multi(tk.Q4_K, [weights[m] for m in names], sizes, ys, x.shape[1], x, M=n)
        return ys

    def _rotate(self, x, pos):
        x = x.view(x.shape[0], -1, self.head_dim)
        half = self.head_dim // 2
        angle = pos[:, None].float() * 10000.0 ** (-torch.arange(half, device="cuda") / half)
        c, s = angle.cos()[:, None], angle.sin()[:, None]
        a, b = x[..., :half], x[..., half:]
        return torch.cat([a * c - b * s, a * s + b * c], -1).flatten(1)

    def forward(self, tokens, q_start, kv_len, pos, max_new):
        """Logits [rows, vocab] of the packed tokens; their keys and values enter the caches."""
        n, D = tokens.numel(), self.head_dim
        assert n <= MAX_ROWS, "one decode step takes up to 16 rows"
        seqs = tk.make_seqs(q_start, kv_len, self.pages, n, max_new)
        norm = lambda h: h * torch.rsqrt(h.square().mean(-1, keepdim=True) + 1e-6)  # noqa: E731
        x = self.embed[tokens.long()]
        for w, cache in zip(self.layers, self.caches):
            q, k, v = self._gemv(["q", "k", "v"], w, norm(x), [self.heads * D, self.kv_heads * D, self.kv_heads * D])
            q, k = self._rotate(q, pos), self._rotate(k, pos)
            self.ctx.kv_append(cache, seqs, k, v)
            a = self.ctx.kv_attend(cache, seqs, q, self.heads, torch.empty_like(q))
            x = x + self._gemv(["o"], w, a, [self.hidden])[0]
            gate, up = self._gemv(["gate", "up"], w, norm(x), [self.ffn, self.ffn])
            x = x + self._gemv(["down"], w, torch.nn.functional.silu(gate) * up, [self.hidden])[0]
        logits = torch.empty(n, self.vocab, device="cuda")
        return self.ctx.gemv(tk.F16, self.head, self.vocab, self.hidden, norm(x), logits, M=n, row_bytes_=2 * self.hidden)


def look_up(text, k):
    """Up to k tokens that followed the last earlier occurrence of the text's last token."""
    for i in range(len(text) - 2, -1, -1):
        if text[i] == text[-1]:
            return text[i + 1:i + 1 + k]
    return []


def generate(model, prompts, steps, drafts=4, temperature=0.0, seed=0):
    """Texts after `steps` steps, and how many drafted tokens were accepted of how many."""
    ctx, B = model.ctx, len(prompts)
    rng = torch.Generator(device="cuda").manual_seed(seed)
    texts = [list(p) for p in prompts]
    for b in range(B):                                   # all but the last token, in steps of up to 16 rows
        for i in range(0, len(texts[b]) - 1, MAX_ROWS):
            part = texts[b][i:min(i + MAX_ROWS, len(texts[b]) - 1)]
            q_start = [0] * (b + 1) + [len(part)] * (B - b)
            kv_len = [i + len(part) if c == b else 1 for c in range(B)]
            model.forward(*_batch(part, q_start, kv_len, range(i, i + len(part))), len(part))
    taken = offered = 0
    for _ in range(steps):
        rows, q_start, kv_len, pos, room = [], [0], [], [], MAX_ROWS // B - 1
        for t in texts:
            d = look_up(t, min(drafts, room))
            offered += len(d)
            rows += [t[-1], *d]
            pos += range(len(t) - 1, len(t) + len(d))
            q_start.append(len(rows))
            kv_len.append(len(t) + len(d))
        tokens, starts, lens, at = _batch(rows, q_start, kv_len, pos)
        logits = model.forward(tokens, starts, lens, at, max(b - a for a, b in zip(q_start, q_start[1:])))
        accepted = torch.empty(B, dtype=torch.int32, device="cuda")
        following = torch.empty(B, dtype=torch.int32, device="cuda")
        ctx.draft_verify(logits, tokens, starts, torch.rand(len(rows), generator=rng, device="cuda"),
                         torch.rand(B, generator=rng, device="cuda"), accepted, following, temperature=temperature)
        for b, (a, x) in enumerate(zip(accepted.tolist(), following.tolist())):
            texts[b] += rows[q_start[b] + 1:q_start[b] + 1 + a] + [x]
            taken += a
    ctx.sync_status()
    return texts, taken, offered


def _batch(rows, q_start, kv_len, pos):
    return tuple(torch.tensor(list(x), dtype=torch.int32, device="cuda") for x in (rows, q_start, kv_len, pos))


def main():
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--steps", type=int, default=40)
    ap.add_argument("--drafts", type=int, default=4)
    ap.add_argument("--temperature", type=float, default=0.0)
    ap.add_argument("--seqs", type=int, default=3)
    a = ap.parse_args()
    ctx = tk.Context()
    model = Decoder(ctx, seqs=a.seqs)
    prompts = [[7 * b + 1, 5, 9 + b, 5, 9 + b, 5] for b in range(a.seqs)]
    texts, taken, offered = generate(model, prompts, a.steps, a.drafts, a.temperature)
    for t in texts:
        print(len(t), "tokens:", t[:24], "...")
    print(f"{taken} of {offered} drafted tokens accepted, {sum(map(len, texts)) / (a.steps * a.seqs):.2f} tokens a step")


if __name__ == "__main__":
    main()
