"""GPU parity of the verification of drafted tokens (tk_draft_verify).

Accepted counts and tokens must equal the plain rule's.  Inputs are kept clear
of its ties: u_accept within 1e-5 of p / q is moved away, so that the rule's
decisions do not turn on the last bit of an exponential; draws are compared
by the interval of the running sum that they hit, 1e-6 wide at most to either
side.  Log-probabilities: 1e-5 absolute (a sum of fp32 terms below 32).
"""
import numpy as np
import pytest

import kv_ref as ref

pytestmark = pytest.mark.gpu


def dev(a):
    import torch
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def softmax(x, T):
    y = x.astype(np.float64) / T
    e = np.exp(y - y.max(-1, keepdims=True))
    return e / e.sum(-1, keepdims=True)


def inputs(seed, rows, V, with_draft, T, sharp=2.0):
    rng = np.random.default_rng(seed)
    start = np.concatenate([[0], np.cumsum(rows)]).astype(np.int32)
    n = int(start[-1])
    target = (rng.standard_normal((n, V)) * sharp).astype(np.float32)
    draft = (target + rng.standard_normal((n, V)) * 0.7).astype(np.float32) if with_draft else None
    tokens = np.zeros(n, np.int32)
    for r in range(n - 1):
        p = softmax(draft[r] if with_draft else target[r] * 2, T or 1.0)
        tokens[r + 1] = rng.choice(V, p=p)
    u = rng.random(n).astype(np.float32)
    if T:                                   # clear of p = u q
        for r in range(n - 1):
            p = softmax(target[r], T)[tokens[r + 1]]
            q = softmax(draft[r], T)[tokens[r + 1]] if with_draft else 1.0
            if abs(u[r] * q - p) < 1e-5 * max(p, q):
                u[r] = np.float32(u[r] * 0.9)
    return start, target, draft, tokens, u, rng.random(len(rows)).astype(np.float32)


def run(ctx, start, target, draft, tokens, ua, us, T, pad=0, logp=True):
    import torch
    B, (n, V) = len(start) - 1, target.shape
    wide = lambda a: None if a is None else dev(np.concatenate([a, np.full((n, pad), 1e9, np.float32)], 1))[:, :V]  # noqa: E731
    acc = torch.full((B,), -7, dtype=torch.int32, device="cuda")
    nxt = torch.full((B,), -7, dtype=torch.int32, device="cuda")
    lp = torch.full((n,), 9.0, device="cuda") if logp else None
    ctx.draft_verify(wide(target), dev(tokens), dev(start), dev(ua), dev(us), acc, nxt, lp, draft=wide(draft), temperature=T)
    torch.cuda.synchronize()
    return acc.cpu().numpy(), nxt.cpu().numpy(), lp.double().cpu().numpy() if logp else None


def check(ctx, got, start, target, draft, tokens, ua, us, T):
    acc, nxt, logp = ref.verify(target, tokens, start, ua, us, draft, T)
    assert np.array_equal(got[0], acc)
    for b in np.flatnonzero(got[1] != nxt):   # only where the draw lies on an edge of the running sum
        r = start[b] + acc[b]
        p = softmax(target[r], T)
        if r < start[b + 1] - 1:
            q = softmax(draft[r], T) if draft is not None else np.eye(1, len(p), tokens[r + 1])[0]
            p = np.maximum(p - q, 0)
        c = np.cumsum(p) / p.sum()
        lo = c[got[1][b] - 1] if got[1][b] else 0.0
        assert lo - 1e-6 <= us[b] <= c[got[1][b]] + 1e-6, b
        logp[r] = got[2][r]
    if got[2] is not None:
        assert np.abs(got[2] - logp).max() < 1e-5


@pytest.mark.parametrize("T", [0.0, 0.5, 1.0, 1.7])
@pytest.mark.parametrize("with_draft", [False, True])
@pytest.mark.parametrize("V", [1, 2, 31, 1000, 4096, 50257])
def test_verify(ctx, T, with_draft, V):
    rows = [1, 5, 2, 8, 3, 1, 9] if V < 50000 else [4, 1, 6]
    for seed in range(2):
        x = inputs(seed + V, rows, V, with_draft, T)
        got = run(ctx, *x, T, pad=seed * 3)
        check(ctx, got, *x, T)
    ctx.sync_status()


@pytest.mark.parametrize("V", [131072, 262144, 300001])
def test_verify_large_vocabulary(ctx, V):
    x = inputs(V, [3, 2], V, True, 0.8, sharp=3.0)
    check(ctx, run(ctx, *x, 0.8), *x, 0.8)
    ctx.sync_status()


@pytest.mark.parametrize("B", [1, 7, 10, 30, 120, 300])
def test_verify_batches_of_every_division(ctx, B):
    """Few sequences are drawn by many thread blocks, many by one each."""
    x = inputs(B, [1 + b % 3 for b in range(B)], 3001, B % 2 == 0, 0.9)
    check(ctx, run(ctx, *x, 0.9), *x, 0.9)
    ctx.sync_status()


@pytest.mark.parametrize("shift", [-3e7, 3e7, -5e6, 1e9])
def test_logits_far_from_zero(ctx, shift):
    """Logits whose exponents pass the packed form's range (2^22): steps of an fp32 there, the same rule."""
    rng = np.random.default_rng(8)
    unit = np.float32(np.spacing(np.float32(abs(shift))))
    t = (np.float32(shift) + unit * rng.integers(-3, 4, (6, 1500)).astype(np.float32)).astype(np.float32)
    start, tokens = np.array([0, 2, 6], np.int32), np.array([0, 7, 0, 8, 9, 10], np.int32)
    ua, us = np.array([0.9, 0.9, 1e-5, 1e-5, 1e-5, 0.5], np.float32), np.array([0.37, 0.81], np.float32)
    for T in (0.0, 1.0):
        acc, nxt, _ = run(ctx, start, t, None, tokens, ua, us, T)
        want = ref.verify(t, tokens, start, ua, us, None, T)
        assert np.array_equal(acc, want[0]) and np.array_equal(nxt, want[1])
    ctx.sync_status()


def test_every_draw_comes_from_its_weights(ctx):
    """8192 draws from one row: the tokens' frequencies fit the residual's within 5 deviations."""
    V, n = 16, 8192
    rng = np.random.default_rng(3)
    t, d = rng.standard_normal((2, V)).astype(np.float32) * 1.5
    start = np.arange(0, 2 * n + 1, 2, dtype=np.int32)
    target, draft = np.tile(t, (2 * n, 1)), np.tile(d, (2 * n, 1))
    x = int((softmax(d, 1.0) / softmax(t, 1.0)).argmax())          # over-drafted: refused with u near 1
    tokens = np.full(2 * n, x, np.int32)
    us = ((np.arange(n) + 0.5) / n).astype(np.float32)
    acc, nxt, _ = run(ctx, start, target, draft, tokens, np.full(2 * n, 0.999999, np.float32), us, 1.0)
    assert (acc == 0).all()
    w = np.maximum(softmax(t, 1.0) - softmax(d, 1.0), 0)
    w /= w.sum()
    seen = np.bincount(nxt, minlength=V) / n
    assert np.abs(seen - w).max() < 1e-3                           # an even grid of draws: one step per edge
    # and the accepted share follows min(1, p / q)
    ua = ((np.arange(2 * n) // 2 + 0.5) / n).astype(np.float32)
    acc, _, _ = run(ctx, start, target, draft, tokens, ua, us, 1.0)
    assert abs(acc.mean() - min(1.0, softmax(t, 1.0)[x] / softmax(d, 1.0)[x])) < 1e-3
    ctx.sync_status()


def test_masked_logits_ties_and_certain_tokens(ctx):
    """-inf and the type's lowest value have no probability; ties go to the lowest token; u = 0; p = q."""
    V = 700
    t = np.full((6, V), -np.inf, np.float32)
    t[0, [5, 9]] = 1.0                       # tie: greedy takes 5
    t[1, 300] = 2.0                          # certain
    t[2, :] = np.finfo(np.float32).min
    t[2, 650] = 0.0
    t[3, [1, 2]] = 0.0
    t[4, [699, 698]] = 3.0
    t[5, :] = 0.0
    start, tokens = np.array([0, 3, 4, 6], np.int32), np.array([0, 5, 300, 0, 0, 698], np.int32)
    ua, us = np.zeros(6, np.float32), np.array([0.5, 0.75, 0.0], np.float32)
    for T in (0.0, 1.0):
        acc, nxt, logp = run(ctx, start, t, None, tokens, ua, us, T)
        assert acc.tolist() == [2, 0, 1]
        assert nxt.tolist() == [650, 1 if T == 0 else 2, 0]
        assert np.allclose(logp, [np.log(0.5), 0, 0, np.log(0.5), np.log(0.5), -np.log(V)], atol=1e-6)
    # draft equal to target: everything is accepted below u = 1, whatever the token
    d = np.random.default_rng(1).standard_normal((6, V)).astype(np.float32)
    u = np.full(6, np.float32(1 - 2.0 ** -24))
    acc, nxt, _ = run(ctx, start, d, d.copy(), np.array([0, 3, 4, 0, 0, 6], np.int32), u, us, 1.0)
    assert acc.tolist() == [2, 0, 1]
    # a drafted token that the target rules out is refused even at u = 0, and never drawn
    t = np.zeros((2, V), np.float32)
    t[:, 7] = -np.inf
    for u0 in (0.0, 0.01, 0.999):
        acc, nxt, _ = run(ctx, np.array([0, 2], np.int32), t, None, np.array([0, 7], np.int32), np.zeros(2, np.float32),
                          np.array([u0], np.float32), 1.0)
        assert acc[0] == 0 and nxt[0] != 7 and 0 <= nxt[0] < V
    # tokens outside the vocabulary are refused
    for bad in (-1, V, 2 ** 31 - 1):
        acc, nxt, _ = run(ctx, np.array([0, 2], np.int32), t, None, np.array([0, bad], np.int32), np.zeros(2, np.float32),
                          np.array([0.5], np.float32), 1.0)
        assert acc[0] == 0 and 0 <= nxt[0] < V
    ctx.sync_status()


def test_rows_without_a_distribution_are_reported(ctx):
    import tier_b200 as tk
    V = 5000
    rng = np.random.default_rng(4)
    base = rng.standard_normal((5, V)).astype(np.float32)
    start, tokens = np.array([0, 3, 5], np.int32), np.zeros(5, np.int32)
    tokens[1:] = base.argmax(1)[:-1]
    ua, us = np.zeros(5, np.float32), np.full(2, 0.5, np.float32)
    for value, T in ((np.nan, 1.0), (np.inf, 0.0), (np.inf, 1.0), (np.nan, 0.0)):
        t = base.copy()
        t[1, 4321] = value
        acc, nxt, logp = run(ctx, start, t, None, tokens, ua, us, T)
        with pytest.raises(tk.TierkError) as e:
            ctx.sync_status()
        assert e.value.status == tk.TK_ERR_DEVICE
        assert acc.tolist() == [1, 1] and nxt[0] == -1 and nxt[1] >= 0 and (logp[1:3] == 0).all()
    t = base.copy()
    t[0] = -np.inf
    acc, nxt, _ = run(ctx, start, t, None, tokens, ua, us, 1.0)
    with pytest.raises(tk.TierkError):
        ctx.sync_status()
    assert nxt[0] == -1 and acc[0] == 0 and nxt[1] >= 0
    # a row that is not needed may hold anything: the last of a draft, and those behind a refusal
    d = base.copy()
    d[[2, 4]] = np.nan
    t = base.copy()
    t[2] = np.nan
    wrong = tokens.copy()
    wrong[1] = int(base[0].argmin())
    u = np.full(5, 0.999, np.float32)
    acc, nxt, _ = run(ctx, start, t, d, wrong, u, us, 1.0)
    ctx.sync_status() if acc[0] == 0 else None
    assert nxt[1] >= 0
    # row_start that does not fit
    for s in ([0, 3, 6], [0, 0, 5], [3, 1, 5], [-1, 3, 5]):
        acc, nxt, _ = run(ctx, np.array(s, np.int32), base, None, tokens, ua, us, 1.0)
        with pytest.raises(tk.TierkError):
            ctx.sync_status()
        assert -1 in nxt


def test_optional_outputs_and_refusals(ctx):
    import torch
    import tier_b200 as tk
    x = inputs(9, [3, 2], 100, True, 1.0)
    a = run(ctx, *x, 1.0)
    b = run(ctx, *x, 1.0, logp=False)
    assert np.array_equal(a[0], b[0]) and np.array_equal(a[1], b[1])
    t, i = torch.zeros(5, 100, device="cuda"), torch.zeros(8, dtype=torch.int32, device="cuda")
    f = torch.zeros(8, device="cuda")
    acc = torch.zeros(2, dtype=torch.int32, device="cuda")
    lib, h = ctx.lib, ctx.h
    p = lambda z: z.data_ptr()  # noqa: E731
    good = [h, 2, p(i), 5, 100, p(t), 100, p(t), 100, p(i), p(f), p(f), 1.0, p(acc), p(acc), None, None]
    for at, value in ((0, None), (1, -1), (2, None), (3, -1), (3, 0), (4, 0), (4, -5), (5, None), (6, 99), (8, 99), (9, None),
                      (10, None), (11, None), (12, -1.0), (12, float("nan")), (12, float("inf")), (12, 1e-6), (13, None), (14, None)):
        args = list(good)
        args[at] = value
        assert lib.tk_draft_verify(*args) == tk.TK_ERR_INVALID, at
        assert b"tk_draft_verify" in lib.tk_last_error_string()
    none = list(good)
    none[1] = 0
    assert lib.tk_draft_verify(*none) == tk.TK_OK
    torch.cuda.synchronize()
    ctx.sync_status()
