"""GPU parity of tk_logprobs and tk_logprobs_grad with plain 64-bit forms
(rows_ref.py holds the forms and the bounds)."""
import math

import pytest

import rows_ref as ref

pytestmark = pytest.mark.gpu
TYPES = ["f32", "f16", "bf16"]


def dt(name):
    import torch
    return {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}[name]


def code(t):
    import tier_b200 as tk
    import torch
    return {torch.float32: tk.DT_F32, torch.float16: tk.DT_F16, torch.bfloat16: tk.DT_BF16}[t.dtype]


def put(t, pad=0, at=0, fill=float("nan")):
    """t's rows on the GPU, `pad` elements apart, the first `at` elements into its memory; `fill` around them."""
    import torch
    n, V = t.shape
    flat = torch.full((n * (V + pad) + at + 8,), fill, dtype=t.dtype, device="cuda")
    view = flat[at:at + n * (V + pad)].view(n, V + pad)[:, :V]
    view.copy_(t)
    return view


def inputs(seed, n, V, dtype, sharp=2.0, hidden=0.0, left=0.0):
    import torch
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(n, V, generator=g) * sharp
    some = torch.randint(V, (n, 4), generator=g)
    x.scatter_add_(1, some, 6 * torch.rand(n, 4, generator=g))
    if hidden:
        x.masked_fill_(torch.rand(n, V, generator=g) < hidden, -math.inf)
        x[:, V // 2] = 1.0
    tokens = torch.where(torch.rand(n, generator=g) < 0.7, some[:, 0], torch.randint(V, (n,), generator=g)).to(torch.int32)
    tokens[torch.rand(n, generator=g) < left] = -1
    return x.to(dt(dtype)), tokens


def forward(ctx, x, tokens, T, k, **kw):
    import torch
    n = x.shape[0]
    out = [torch.full((n,), 7.0, device="cuda") for _ in range(4)]
    ids = torch.full((n, k), 7, dtype=torch.int32, device="cuda") if k else None
    lp = torch.full((n, k), 7.0, device="cuda") if k else None
    tokens = tokens.cuda() if tokens is not None else None
    ctx.logprobs(x, tokens, out[0] if tokens is not None else None, out[1], out[2], out[3], ids, lp, temperature=T,
                 x_dtype=code(x), **kw)
    if tokens is None:
        out[0] = None
    return out + ([ids, lp] if k else [])


def check(got, want, tol):
    import torch
    for i, (g, w, t) in enumerate(zip(got, want, tol)):
        if g is None:
            continue
        g = g.cpu()
        if t is None:
            assert torch.equal(g.long(), w.long()), (i, (g.long() != w.long()).nonzero()[:5])
            continue
        g = g.double()
        same = (g == w) | (g.isnan() & w.isnan())
        off = ((g - w).abs() / t.clamp(min=1e-300)).masked_fill(same, 0.0)
        assert (off <= 1).all(), (i, off.max(), off.argmax(), g.flatten()[off.argmax()], w.flatten()[off.argmax()])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("V", [1, 2, 7, 31, 255, 1000, 4096, 8193, 50257])
def test_rows_of_every_size(ctx, V, dtype):
    for seed, (n, T, k, pad, at) in enumerate([(1, 1.0, 1, 0, 0), (3, 0.6, 5, 1, 3), (17, 2.5, 64, 8, 1), (5, 1.0, 256, 5, 7),
                                               (40, 1.0, 0, 3, 2)]):
        k = min(k, V)
        x, tokens = inputs(seed + V, n, V, dtype, left=0.2 * (seed > 1))
        got = forward(ctx, put(x, pad, at), tokens, T, k)
        check(got, *ref.logprobs(x, tokens, T, k))
    ctx.sync_status()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n", [1, 2, 5, 9, 20, 37, 80, 150, 300])
def test_batches_of_every_division(ctx, n, dtype):
    """Few rows are cut into many parts, many rows into few."""
    for V, k in ((20001, 20), (65536, 3)):
        if n * V > 1 << 23:
            continue
        x, tokens = inputs(n, n, V, dtype, left=0.1)
        check(forward(ctx, put(x, n % 3), tokens, 1.0, k), *ref.logprobs(x, tokens, 1.0, k))
    ctx.sync_status()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,k", [(1, 20), (1, 256), (3, 128), (30, 7)])
def test_large_vocabulary(ctx, n, k, dtype):
    for V in (131072, 262144, 300001):
        x, tokens = inputs(V + n, n, V, dtype)
        check(forward(ctx, put(x, V % 2), tokens, 0.8, k), *ref.logprobs(x, tokens, 0.8, k))
    ctx.sync_status()


def test_largest_vocabulary(ctx):
    import torch
    V = 1 << 23
    for dtype, n, k in (("f32", 1, 256), ("bf16", 2, 64), ("bf16", 400, 5)):
        g = torch.Generator(device="cuda").manual_seed(n)
        x = torch.empty(n, V, dtype=dt(dtype), device="cuda")
        for i in range(n):
            x[i] = (torch.randn(V, generator=g, device="cuda") * 2).to(x.dtype)
        tokens = torch.arange(n, dtype=torch.int32) * 1000 + V // 2
        got = forward(ctx, x, tokens, 1.0, k)
        some = [0, n // 2, n - 1]
        want, tol = ref.logprobs(x[some].cpu(), tokens[some], 1.0, k)
        check([t[some] for t in got], want, tol)
        del x
    ctx.sync_status()


@pytest.mark.parametrize("dtype", TYPES)
def test_orders_and_ties(ctx, dtype):
    """Rows whose largest logits stand where they are hard to find: all alike, rising, falling, in one place, few values."""
    import tier_b200 as tk
    import torch
    V = 70001
    i = torch.arange(V, dtype=torch.float64)
    g = torch.Generator().manual_seed(5)
    rows = [torch.zeros(V), torch.full((V,), -3.4e38 if dtype != "f16" else -65504.0), i / V * 20, -i / V * 20,
            torch.randint(0, 3, (V,), generator=g).double(), torch.randn(V, generator=g).double().round(),
            torch.where(i % 2 == 0, 0.0, -0.0), torch.where(i > V - 400, 5.0 + i / V, 0.0), torch.where(i < 300, 5.0, i / V),
            torch.where(i % 997 == 3, 4.0, -2.0), torch.full((V,), -math.inf).index_fill(0, torch.tensor([9, 40000, V - 1]), 2.0),
            torch.where(i == V - 1, 1e4, -1e4), torch.where(i % 4096 < 3, 3.0, 0.0), i.remainder(8192) / 8192]
    x = torch.stack([r.double() for r in rows]).to(dt(dtype))
    for n in (len(rows), 300):                       # few parts and many
        y = x.repeat((n + len(rows) - 1) // len(rows), 1)[:n] if n > len(rows) else x
        tokens = (torch.arange(n, dtype=torch.int32) * 31) % 300
        for k in (1, 17, 256):
            got = forward(ctx, put(y, 1), tokens, 1.0, k)
            want, tol = ref.logprobs(x, tokens[:len(rows)], 1.0, k)
            check([t[:len(rows)] for t in got], want, tol)
            if n > len(rows):                        # the same rows again: the same lists
                assert torch.equal(got[4][len(rows):2 * len(rows)], got[4][:len(rows)])
    if not ref.without(x).any():                     # (bf16 rounds -3.4e38 to -inf: a row of nothing, which is reported)
        return ctx.sync_status()
    with pytest.raises(tk.TierkError):
        ctx.sync_status()


@pytest.mark.parametrize("dtype", TYPES)
def test_masks(ctx, dtype):
    """-inf and the type's lowest value in places of the row; the only logit that is left."""
    import torch
    x, tokens = inputs(3, 12, 5003, dtype, hidden=0.5)
    x[4] = torch.where(x[4] == -math.inf, torch.finfo(x.dtype).min, x[4])
    x[5] = torch.finfo(x.dtype).min
    x[5, 77] = torch.finfo(x.dtype).max
    x[6, :] = -math.inf
    x[6, 5002] = -3.0
    tokens[6] = 5002
    x[7] = torch.finfo(x.dtype).max
    tokens[8] = int((x[8] == -math.inf).nonzero()[0])     # an impossible token: -inf
    for T in (1.0, 1e-4, 1e4):
        got = forward(ctx, put(x, 1, 1), tokens, T, 20)
        want, tol = ref.logprobs(x, tokens, T, 20)
        check(got, want, tol)
    assert got[0][8] == -math.inf
    ctx.sync_status()


@pytest.mark.parametrize("n", [6, 700])
def test_rows_that_hold_no_distribution(ctx, n):
    """NaN, +inf, only -inf: NaN and -1 in their rows, and the status; rows left out are not looked at."""
    import tier_b200 as tk
    import torch
    x, tokens = inputs(7, n, 9001, "f32")
    bad = {0: math.nan, 2: math.inf, 4: -math.inf}
    x[0, 8999], x[2, 0], x[4] = math.nan, math.inf, -math.inf
    x[1], tokens[1] = math.nan, -1
    got = [t.cpu() for t in forward(ctx, put(x), tokens, 1.0, 4)]
    with pytest.raises(tk.TierkError) as e:
        ctx.sync_status()
    assert e.value.status == tk.TK_ERR_DEVICE
    for r in bad:
        assert all(t[r].isnan().all() for t in got[:4] + got[5:]) and (got[4][r] == -1).all()
    good = torch.tensor([i for i in range(n) if i not in bad])
    want, tol = ref.logprobs(x[good].nan_to_num(0.0), tokens[good], 1.0, 4)
    check([t[good] for t in got], want, tol)
    ctx.sync_status()
    x[0], x[2], x[4], tokens[3] = 0.0, 0.0, 0.0, 9001     # beyond the vocabulary: left out, reported
    got = forward(ctx, put(x), tokens, 1.0, 4)
    with pytest.raises(tk.TierkError):
        ctx.sync_status()
    check(got, *ref.logprobs(x.nan_to_num(0.0), tokens, 1.0, 4))


def test_outputs_are_optional(ctx):
    import torch
    x, tokens = inputs(2, 9, 3001, "bf16")
    gx = put(x)
    want, tol = ref.logprobs(x, tokens, 1.0, 6)
    check(forward(ctx, gx, None, 1.0, 6), *ref.logprobs(x, None, 1.0, 6))
    lp = torch.zeros(9, device="cuda")
    ctx.logprobs(gx, tokens.cuda(), lp, x_dtype=code(gx))
    check([lp], want[:1], tol[:1])
    ids = torch.zeros(9, 6, dtype=torch.int32, device="cuda")
    ctx.logprobs(gx, top_ids=ids, x_dtype=code(gx))
    check([ids], want[4:5], [None])
    ctx.logprobs(gx[:0], tokens.cuda()[:0], lp, x_dtype=code(gx))
    ctx.sync_status()


def gradient(ctx, x, tokens, T, d_logp, d_entropy, dtype, out=None, pad=0, at=0):
    import torch
    fw = forward(ctx, x, tokens, T, 0)
    dx = put(torch.full(x.shape, 7.0, dtype=dt(dtype)), pad, at, 7.0) if out is None else out
    cu = lambda t: None if t is None else t.cuda()  # noqa: E731
    ctx.logprobs_grad(x, cu(tokens), fw[2], fw[3], dx, cu(d_logp), fw[1], cu(d_entropy), temperature=T, x_dtype=code(x),
                      d_dtype=code(dx))
    return dx


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d", TYPES)
@pytest.mark.parametrize("V", [1, 2, 13, 1000, 8193, 50257])
def test_gradient(ctx, V, dtype, d):
    import torch
    for seed, (n, T, pad, at, pad2, at2) in enumerate([(1, 1.0, 0, 0, 0, 0), (7, 0.6, 1, 3, 1, 3), (19, 2.5, 8, 1, 0, 0),
                                                       (4, 1.0, 0, 0, 3, 5)]):
        x, tokens = inputs(seed + V, n, V, dtype, left=0.2 * (seed > 1), hidden=0.1 * (seed == 1))
        g = torch.Generator().manual_seed(seed)
        dl, de = torch.randn(n, generator=g), 0.1 * torch.randn(n, generator=g)
        for a, b in ((dl, de), (dl, None), (None, de)):
            dx = gradient(ctx, put(x, pad, at), tokens, T, a, b, d, pad=pad2, at=at2)
            want, tol = ref.logprobs_grad(x, tokens, T, a, b, dt(d))
            check([dx], [want], [tol])
            if pad2:                                  # nothing beside the rows is written
                around = dx.as_strided((n, V + pad2), (V + pad2, 1))[:-1, V:]
                assert (around == 7.0).all()
    ctx.sync_status()


def test_gradient_against_differences(ctx):
    """d/dl of sum_i (a_i logp_i + b_i entropy_i) by differences of the forward pass in 64 bits."""
    import torch
    x, tokens = inputs(1, 3, 50, "f32")
    a, b, T = torch.tensor([1.0, -0.5, 0.0]), torch.tensor([0.3, 0.0, -1.0]), 1.3
    dx = gradient(ctx, put(x), tokens, T, a, b, "f32").cpu().double()

    def total(z):
        lp = torch.log_softmax(z / T, 1)
        return (a.double() * lp.gather(1, tokens.long()[:, None])[:, 0] - b.double() * (lp.exp() * lp).sum(1)).sum()

    h = 1e-5
    for r in range(3):
        for j in range(0, 50, 7):
            e = torch.zeros_like(x, dtype=torch.float64)
            e[r, j] = h
            slope = (total(x.double() + e) - total(x.double() - e)) / (2 * h)
            assert abs(slope - dx[r, j]) < 2e-6           # differences: h^2 and 2^-52 / h


@pytest.mark.parametrize("dtype", TYPES)
def test_gradient_in_place(ctx, dtype):
    import torch
    for n, V, pad in ((3, 9001, 2), (200, 1001, 0)):
        x, tokens = inputs(4, n, V, dtype, left=0.1)
        dl, de = torch.linspace(-1, 1, n), torch.full((n,), 0.05)
        view = put(x, pad, 1)
        gradient(ctx, view, tokens, 1.0, dl, de, dtype, out=view)
        want, tol = ref.logprobs_grad(x, tokens, 1.0, dl, de, dt(dtype))
        check([view], [want], [tol])
        both = torch.zeros(n, 2 * V + 3, dtype=dt(dtype), device="cuda")       # columns of one matrix
        both[:, :V] = x
        gradient(ctx, both[:, :V], tokens, 1.0, dl, de, dtype, out=both[:, V + 2:2 * V + 2])
        check([both[:, V + 2:2 * V + 2]], [want], [tol])
        assert torch.equal(both[:, :V].cpu(), x) and (both[:, V:V + 2] == 0).all() and (both[:, 2 * V + 2:] == 0).all()
    ctx.sync_status()


def test_rows_without_gradient_are_not_read(ctx):
    import torch
    x, tokens = inputs(6, 5, 4001, "bf16")
    x[1], x[3] = math.nan, math.nan
    tokens[1] = -1
    gx, one = put(x), torch.ones(5)
    dl = torch.tensor([1.0, 2.0, 0.5, 0.0, 1.0]).cuda()
    dx = torch.full((5, 4001), 7.0, device="cuda")
    fw = forward(ctx, put(x.nan_to_num(0.0)), tokens, 1.0, 0)
    ctx.logprobs_grad(gx, tokens.cuda(), fw[2], fw[3], dx, dl, x_dtype=code(gx), d_dtype=0)
    ctx.sync_status()
    want, tol = ref.logprobs_grad(x.nan_to_num(0.0), tokens, 1.0, dl.cpu(), None, torch.float32)
    check([dx], [want], [tol])
    assert (dx[1] == 0).all() and (dx[3] == 0).all() and one.sum() == 5


def test_rows_beyond_32_bits(ctx):
    """Rows 2^29 elements apart: places past 2^31 elements and 2^32 bytes."""
    import torch
    V, ld, n = 1009, (1 << 29) + 1, 6
    flat = torch.zeros((n - 1) * ld + V, dtype=torch.bfloat16, device="cuda")
    view = flat.as_strided((n, V), (ld, 1))
    x, tokens = inputs(9, n, V, "bf16")
    view.copy_(x)
    check(forward(ctx, view, tokens, 1.0, 9), *ref.logprobs(x, tokens, 1.0, 9))
    gradient(ctx, view, tokens, 1.0, torch.ones(n), None, "bf16", out=view)
    want, tol = ref.logprobs_grad(x, tokens, 1.0, torch.ones(n), None, torch.bfloat16)
    check([view], [want], [tol])
    flat[torch.arange(n, device="cuda")[:, None] * ld + torch.arange(V, device="cuda")[None]] = 0
    assert not flat.any()
    ctx.sync_status()


def test_captured_and_on_another_stream(ctx):
    """One graph of forward and gradient, replayed with other contents; a call on a stream that is not the current one."""
    import torch
    x, tokens = inputs(1, 10, 20011, "bf16")
    gx, tk_ = put(x), tokens.cuda()
    f = [torch.zeros(10, device="cuda") for _ in range(4)]
    ids = torch.zeros(10, 8, dtype=torch.int32, device="cuda")
    lp, dx, one = torch.zeros(10, 8, device="cuda"), torch.zeros_like(gx), torch.ones(10, device="cuda")

    def step():
        ctx.logprobs(gx, tk_, *f, ids, lp, x_dtype=code(gx))
        ctx.logprobs_grad(gx, tk_, f[2], f[3], dx, one, f[1], one, x_dtype=code(gx))

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for seed in (2, 3):
        x, tokens = inputs(seed, 10, 20011, "bf16", left=0.3)
        gx.copy_(x)
        tk_.copy_(tokens)
        graph.replay()
        torch.cuda.synchronize()
        check(f + [ids, lp], *ref.logprobs(x, tokens, 1.0, 8))
        want, tol = ref.logprobs_grad(x, tokens, 1.0, torch.ones(10), torch.ones(10), torch.bfloat16)
        check([dx], [want], [tol])
        ids.zero_()
        dx.zero_()
        torch.cuda.synchronize()
        ctx.logprobs(gx, tk_, *f, ids, lp, x_dtype=code(gx), stream=side)
        side.synchronize()
        check(f + [ids, lp], *ref.logprobs(x, tokens, 1.0, 8))
    ctx.sync_status()


def test_the_same_again_is_the_same(ctx):
    """No result depends on an order of arrival."""
    import torch
    x, tokens = inputs(8, 37, 50257, "f32")
    gx = put(x)
    first = forward(ctx, gx, tokens, 0.9, 40)
    for _ in range(5):
        assert all(torch.equal(a, b) for a, b in zip(first, forward(ctx, gx, tokens, 0.9, 40)))


def test_refusals(ctx):
    import tier_b200 as tk
    import torch
    x, v = torch.zeros(4, 100, device="cuda"), torch.zeros(4, device="cuda")
    tok = torch.zeros(4, dtype=torch.int32, device="cuda")
    wide, ids = torch.zeros(4, 400, device="cuda"), torch.zeros(4, 101, dtype=torch.int32, device="cuda")

    def refused(what, fn, *a, status=tk.TK_ERR_INVALID, **kw):
        with pytest.raises(tk.TierkError) as e:
            fn(*a, **kw)
        assert e.value.status == status and what in str(e.value), str(e.value)

    refused("no tokens", ctx.logprobs, x, None, v)
    refused("top_k", ctx.logprobs, x, tok, v, top_ids=ids)                       # more than the vocabulary
    refused("top_k", ctx.logprobs, wide, tok, v, top_ids=torch.zeros(4, 257, dtype=torch.int32, device="cuda"))
    refused("do not fit", ctx.logprobs, x, tok, v, top_logp=v)
    for T in (0.0, -1.0, math.nan, math.inf, 1e-5, 1e5):
        refused("temperature", ctx.logprobs, x, tok, v, temperature=T)
    refused("unknown element type", ctx.logprobs, x, tok, v, x_dtype=9)
    lib, p = ctx.lib, lambda t: t.data_ptr()  # noqa: E731
    s = torch.cuda.current_stream().cuda_stream

    def raw(n=4, V=100, xp=p(x), xt=0, ld=100, T=1.0):
        return lib.tk_logprobs(ctx.h, n, V, xp, xt, ld, p(tok), T, p(v), None, None, None, 0, None, None, s)

    assert raw() == tk.TK_OK and raw(n=0, xp=None) == tk.TK_OK
    assert raw(n=-1) == tk.TK_ERR_INVALID and raw(V=0) == tk.TK_ERR_INVALID and raw(ld=99) == tk.TK_ERR_INVALID
    assert raw(xp=None) == tk.TK_ERR_INVALID and raw(xp=p(x) + 2) == tk.TK_ERR_INVALID and raw(xt=3) == tk.TK_ERR_INVALID
    assert raw(V=(1 << 23) + 1, ld=1 << 24) == tk.TK_ERR_UNSUPPORTED and raw(ld=1 << 62) == tk.TK_ERR_INVALID
    refused("neither gradient", ctx.logprobs_grad, x, tok, v, v, torch.zeros_like(x))
    refused("no tokens", ctx.logprobs_grad, x, None, v, v, torch.zeros_like(x), v)
    refused("needs the entropy", ctx.logprobs_grad, x, tok, v, v, torch.zeros_like(x), v, None, v)
    refused("null pointer", ctx.logprobs_grad, x, tok, None, v, torch.zeros_like(x), v)
    refused("overlaps", ctx.logprobs_grad, wide[:, :100], tok, v, v, wide[:, 99:199], v)
    refused("overlaps", ctx.logprobs_grad, wide[:, :100], tok, v, v, wide[:, 1:101], v)
    refused("overlaps", ctx.logprobs_grad, wide[:3, 350:], tok, v, v,
            wide.as_strided((3, 50), (400, 1), 380), v)
    refused("overlaps", ctx.logprobs_grad, x, tok, v, v, x.view(torch.bfloat16)[:, :100], v, d_dtype=tk.DT_BF16)
    ctx.logprobs_grad(wide[:, :100], tok, v, v + 1, wide[:, 100:200], v)
    ctx.sync_status()
