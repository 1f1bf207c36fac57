"""GPU parity of tk_distill and tk_distill_grad with plain 64-bit forms
(rows_ref.py holds the forms and the bounds), and the run of a teacher, a
student and the LM head's products around them."""
import math

import pytest

import rows_ref as ref
from test_gpu_logprobs import TYPES, check, code, dt, put

pytestmark = pytest.mark.gpu


def inputs(seed, n, V, k, dtype, short=0.2, empty=0.1, twice=0.0, hidden=0.0):
    import torch
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(n, V, generator=g) * 2
    some = torch.randint(V, (n, 4), generator=g)
    x.scatter_add_(1, some, 6 * torch.rand(n, 4, generator=g))
    if hidden:
        x.masked_fill_(torch.rand(n, V, generator=g) < hidden, -math.inf)
        x[:, V // 2] = 1.0
    ids = torch.stack([torch.randperm(V, generator=g)[torch.arange(k) % V] for _ in range(n)])
    if twice:
        ids = torch.where(torch.rand(n, k, generator=g) < twice, ids[:, :1], ids)
    ids[torch.rand(n, k, generator=g) < short] = -1
    ids[torch.rand(n, generator=g) < empty] = -1
    t = torch.randn(n, k, generator=g) * 2
    return x.to(dt(dtype)), ids.to(torch.int32), t, torch.rand(n, generator=g) + 0.5


def run(ctx, x, ids, t, T, weight, dx=None, **kw):
    """loss, rmax, rsum (and dlogits)."""
    import torch
    out = [torch.full((x.shape[0],), 7.0, device="cuda") for _ in range(3)]
    grad = {} if dx is None else {"dlogits": dx, "d_dtype": code(dx)}
    if weight is not None:
        grad["weight"] = weight.cuda()
    ctx.distill(x, ids.cuda(), t.cuda(), out[0], rmax=out[1], rsum=out[2], temperature=T, x_dtype=code(x), **grad, **kw)
    return out + ([] if dx is None else [dx])


def blank(x, dtype, pad=0, at=0):
    import torch
    return put(torch.full(x.shape, 7.0, dtype=dt(dtype)), pad, at, 7.0)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d", TYPES)
@pytest.mark.parametrize("V", [1, 2, 13, 1000, 8193, 50257])
def test_loss_and_gradient(ctx, V, dtype, d):
    for seed, (n, k, T, pad, at, pad2, at2) in enumerate([(1, 1, 1.0, 0, 0, 0, 0), (7, 5, 2.0, 1, 3, 1, 3),
                                                          (19, 64, 0.7, 8, 1, 0, 0), (4, 256, 1.0, 0, 0, 3, 5)]):
        x, ids, t, w = inputs(seed + V, n, V, k, dtype, twice=0.3 * (seed == 2), empty=0.2 * (seed > 0))
        want, tol = ref.distill(x, ids, t, T, w, dt(d))
        gx = put(x, pad, at)
        got = run(ctx, gx, ids, t, T, w, blank(x, d, pad2, at2))
        check(got, want, tol)
        check(run(ctx, gx, ids, t, T, w), want[:3], tol[:3])           # the loss alone
        dx = blank(x, d, pad2, at2)
        ctx.distill_grad(gx, ids.cuda(), t.cuda(), got[1], got[2], dx, w.cuda(), temperature=T, x_dtype=code(gx), d_dtype=code(dx))
        check([dx], want[3:], tol[3:])
        if pad2:
            for o in (dx, got[3]):
                assert (o.as_strided((n, V + pad2), (V + pad2, 1))[:-1, V:] == 7.0).all()
    ctx.sync_status()


@pytest.mark.parametrize("n", [1, 2, 5, 9, 20, 37, 80, 150, 300])
def test_batches_of_every_division(ctx, n):
    for V, dtype, d in ((20001, "f32", "bf16"), (65536, "bf16", "bf16"), (30000, "f16", "f32")):
        if n * V > 1 << 23:
            continue
        x, ids, t, w = inputs(n, n, V, 20, dtype)
        want, tol = ref.distill(x, ids, t, 1.0, None, dt(d))
        check(run(ctx, put(x), ids, t, 1.0, None, blank(x, d)), want, tol)
    ctx.sync_status()


@pytest.mark.parametrize("dtype,d", [("f32", "f32"), ("f32", "bf16"), ("bf16", "bf16"), ("f16", "f32")])
def test_large_vocabulary(ctx, dtype, d):
    for V, n in ((262144, 3), (300001, 2), (1 << 20, 1)):
        x, ids, t, w = inputs(V, n, V, 100, dtype, empty=0.0)
        want, tol = ref.distill(x, ids, t, 2.0, w, dt(d))
        got = run(ctx, put(x), ids, t, 2.0, w, blank(x, d))
        check(got, want, tol)
        dx = blank(x, d)
        ctx.distill_grad(put(x), ids.cuda(), t.cuda(), got[1], got[2], dx, w.cuda(), temperature=2.0, x_dtype=code(x),
                         d_dtype=code(dx))
        check([dx], want[3:], tol[3:])
    ctx.sync_status()


def test_largest_vocabulary(ctx):
    x, ids, t, w = inputs(1, 1, 1 << 23, 256, "bf16", empty=0.0)
    want, tol = ref.distill(x, ids, t, 1.0, w, dt("bf16"))
    check(run(ctx, put(x), ids, t, 1.0, w, blank(x, "bf16")), want, tol)
    ctx.sync_status()


@pytest.mark.parametrize("dtype", TYPES)
def test_in_place(ctx, dtype):
    import torch
    for n, V, pad, k in ((3, 9001, 2, 30), (200, 1001, 0, 256), (2, 262144, 0, 50)):
        x, ids, t, w = inputs(n, n, V, k, dtype, twice=0.2)
        want, tol = ref.distill(x, ids, t, 1.0, w, dt(dtype))
        view = put(x, pad, 1)
        check(run(ctx, view, ids, t, 1.0, w, view), want, tol)
        other = put(x, pad, 1)
        st = run(ctx, other, ids, t, 1.0, w)
        ctx.distill_grad(other, ids.cuda(), t.cuda(), st[1], st[2], other, w.cuda(), x_dtype=code(other))
        check([other], want[3:], tol[3:])
    assert torch.isfinite(view).all()
    ctx.sync_status()


@pytest.mark.parametrize("dtype", TYPES)
def test_masks(ctx, dtype):
    """Forbidden tokens in the student's rows and the teacher's lists, lowest values, a teacher certain of one token."""
    import torch
    x, ids, t, w = inputs(3, 10, 5003, 30, dtype, hidden=0.4, short=0.0, empty=0.0)
    x[4] = torch.where(x[4] == -math.inf, torch.finfo(x.dtype).min, x[4])
    x[5] = torch.finfo(x.dtype).min
    x[5, 77] = torch.finfo(x.dtype).max
    t[6], t[6, 3] = -math.inf, 2.0                       # one entry left
    t[7] = -math.inf                                     # none: as without entries
    t[8] = torch.where(torch.arange(30) % 2 == 0, -3.4e38, 3.4e38)
    t[9] = torch.linspace(0, -300, 30)
    ids[9] = torch.arange(30)
    x[9, :20], x[9, 20:30] = 0.5, -math.inf              # q is 0 where p is
    for T in (1.0, 0.3, 3.0):
        want, tol = ref.distill(x, ids, t, T, w, torch.float32)
        got = run(ctx, put(x, 1), ids, t, T, w, blank(x, "f32"))
        assert (want[0] == math.inf).any()
        check(got, want, tol)
    assert (got[3][7] == 0).all() and got[0][7] == 0
    ctx.sync_status()


@pytest.mark.parametrize("n", [8, 700])
def test_rows_that_hold_no_distribution(ctx, n):
    import tier_b200 as tk
    import torch
    x, ids, t, w = inputs(7, n, 9001, 10, "f32", empty=0.0, short=0.0)
    x[0, 8999], x[2, 0], x[4], t[5, 3], t[6, 0] = math.nan, math.inf, -math.inf, math.nan, math.inf
    bad = [0, 2, 4, 5, 6]
    x[1], ids[1] = math.nan, -1                          # not looked at
    w[4] = 0.0                                           # no gradient, whatever the row holds
    dx = blank(x, "f32")
    got = [g.cpu() for g in run(ctx, put(x), ids, t, 1.0, w, dx)]
    with pytest.raises(tk.TierkError) as e:
        ctx.sync_status()
    assert e.value.status == tk.TK_ERR_DEVICE
    for r in bad:
        assert all(o[r].isnan() for o in got[:3]) and (got[3][r] == 0 if r == 4 else got[3][r].isnan()).all()
    good = torch.tensor([i for i in range(n) if i not in bad])
    want, tol = ref.distill(x[good].nan_to_num(0.0), ids[good], t[good], 1.0, w[good], torch.float32)
    check([g[good] for g in got], want, tol)
    ctx.sync_status()
    # a place beyond the vocabulary does not count, and is reported
    x, ids, t, w = inputs(7, n, 9001, 10, "f32")
    ids[3, 4], ids[2, 0] = 9001, 2 ** 31 - 1
    got = run(ctx, put(x), ids, t, 1.0, w, dx)
    with pytest.raises(tk.TierkError):
        ctx.sync_status()
    check(got, *ref.distill(x, ids, t, 1.0, w, torch.float32))
    ctx.distill_grad(put(x), ids.cuda(), t.cuda(), got[1], got[2], dx, w.cuda())
    with pytest.raises(tk.TierkError):
        ctx.sync_status()
    check([dx], *[[v[3]] for v in ref.distill(x, ids, t, 1.0, w, torch.float32)])


def test_gradient_against_differences(ctx):
    import torch
    x, ids, t, w = inputs(1, 3, 50, 6, "f32", empty=0.0, twice=0.3)
    T = 1.7
    dx = run(ctx, put(x), ids, t, T, w, blank(x, "f32"))[3].cpu().double()

    def total(z):
        return (ref.distill(z, ids, t, T, None, None)[0][0] * w.double()).sum()

    h = 1e-5
    for r in range(3):
        for j in list(range(0, 50, 9)) + [i for i in ids[r].tolist() if i >= 0]:
            e = torch.zeros_like(x, dtype=torch.float64)
            e[r, j] = h
            slope = (total(x.double() + e) - total(x.double() - e)) / (2 * h)
            assert abs(slope - dx[r, j]) < 2e-6


def test_captured_and_on_another_stream(ctx):
    import torch
    x, ids, t, w = inputs(1, 12, 20011, 16, "bf16")
    gx, gi, gt, gw = put(x), ids.cuda(), t.cuda(), w.cuda()
    out, dx, dx2 = [torch.zeros(12, device="cuda") for _ in range(3)], torch.zeros_like(gx), torch.zeros_like(gx)

    def step(**kw):
        ctx.distill(gx, gi, gt, out[0], gw, dx, out[1], out[2], x_dtype=code(gx), **kw)
        ctx.distill_grad(gx, gi, gt, out[1], out[2], dx2, gw, x_dtype=code(gx), **kw)

    side = torch.cuda.Stream()
    step(stream=side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for seed in (2, 3):
        x, ids, t, w = inputs(seed, 12, 20011, 16, "bf16")
        for a, b in ((gx, x), (gi, ids), (gt, t), (gw, w)):
            a.copy_(b)
        graph.replay()
        torch.cuda.synchronize()
        want, tol = ref.distill(x, ids, t, 1.0, w, torch.bfloat16)
        check(out + [dx], want, tol)
        check([dx2], want[3:], tol[3:])
    first = [o.clone() for o in out + [dx]]
    for _ in range(4):
        step()
        assert all(torch.equal(a, b) for a, b in zip(first, out + [dx]))
    ctx.sync_status()


def test_rows_beyond_32_bits(ctx):
    import torch
    V, ld, n = 1009, (1 << 29) + 1, 6
    flat = torch.zeros((n - 1) * ld + V, dtype=torch.bfloat16, device="cuda")
    view = flat.as_strided((n, V), (ld, 1))
    x, ids, t, w = inputs(9, n, V, 9, "bf16")
    view.copy_(x)
    want, tol = ref.distill(x, ids, t, 1.0, w, torch.bfloat16)
    check(run(ctx, view, ids, t, 1.0, w, view), want, tol)
    flat[torch.arange(n, device="cuda")[:, None] * ld + torch.arange(V, device="cuda")[None]] = 0
    assert not flat.any()
    ctx.sync_status()


def test_refusals(ctx):
    import tier_b200 as tk
    import torch
    x, v = torch.zeros(4, 100, device="cuda"), torch.zeros(4, device="cuda")
    ids, t = torch.zeros(4, 5, dtype=torch.int32, device="cuda"), torch.zeros(4, 5, device="cuda")

    def refused(what, fn, *a, **kw):
        with pytest.raises(tk.TierkError) as e:
            fn(*a, **kw)
        assert e.value.status == tk.TK_ERR_INVALID and what in str(e.value), str(e.value)

    big = torch.zeros(4, 257, dtype=torch.int32, device="cuda")
    refused("k must be", ctx.distill, x, big, torch.zeros(4, 257, device="cuda"), v)
    refused("k must be", ctx.distill, x, ids[:, :0], t[:, :0], v)
    refused("null pointer", ctx.distill, x, ids, None, v)
    refused("matrix of 4 rows", ctx.distill, x, ids[:3], t, v)
    refused("contiguous", ctx.distill, x, big[:, :5], t, v)
    refused("temperature", ctx.distill, x, ids, t, v, temperature=0.0)
    refused("overlaps", ctx.distill, x, ids, t, v, dlogits=x.view(torch.bfloat16).view(-1).as_strided((4, 100), (101, 1), 3),
            d_dtype=tk.DT_BF16)
    refused("unknown element type", ctx.distill, x, ids, t, v, dlogits=torch.zeros_like(x), d_dtype=5)
    refused("null pointer", ctx.distill_grad, x, ids, t, None, v, torch.zeros_like(x))
    refused("null pointer", ctx.distill_grad, x, ids, t, v, v, None)
    assert ctx.lib.tk_distill(ctx.h, 0, 100, None, 0, 100, 5, None, None, 1.0, None, None, None, None, None, 0, 0, None) == tk.TK_OK
    assert ctx.lib.tk_distill(ctx.h, -1, 100, None, 0, 100, 5, None, None, 1.0, None, None, None, None, None, 0, 0, None) == 1
    ctx.distill(x[:0], ids[:0], t[:0], v)
    ctx.sync_status()


def test_a_step_of_distillation(ctx):
    """Teacher's head -> its top tokens -> student's head -> loss and gradient -> the head's input gradient, against 64 bits."""
    import tier_b200 as tk
    import torch
    n, V, H, k, T = 200, 5000, 256, 40, 2.0
    g = torch.Generator().manual_seed(0)
    heads = [(torch.randn(V, H, generator=g) * 0.1).half() for _ in range(2)]
    hidden = [torch.randn(n, H, generator=g) for _ in range(2)]
    W = [tk.make_weight(tk.F16, V, H, h.cuda()) for h in heads]
    logits = [torch.empty(n, V, device="cuda") for _ in range(2)]
    for i in range(2):
        ctx.linear(W[i], hidden[i].cuda(), n, logits[i])
    ids, lp = torch.empty(n, k, dtype=torch.int32, device="cuda"), torch.empty(n, k, device="cuda")
    ctx.logprobs(logits[0], top_ids=ids, top_logp=lp)
    loss, dX = torch.empty(n, device="cuda"), torch.empty(n, H, device="cuda")
    weight = torch.full((n,), 1.0 / n, device="cuda")
    ctx.distill(logits[1], ids, lp, loss, weight, logits[1], temperature=T)       # in place: the logits are not needed again
    ctx.linear_dx(W[1], logits[1], n, dX)
    ctx.sync_status()
    exact = [h.double() @ w.double().T for h, w in zip(hidden, heads)]
    top = exact[0].topk(k, dim=1)
    assert (ids.cpu().long() == top.indices).float().mean() > 0.999              # (logits of 1e-5 apart may change places)
    want, _ = ref.distill(exact[1], ids.cpu(), torch.log_softmax(exact[0], 1).gather(1, ids.cpu().long()), T, weight.cpu(),
                          torch.float32)
    # the heads' products are within 1e-5 of their rows' size (up to 8 here); losses and gradients follow them
    assert (loss.cpu().double() - want[0]).abs().max() < 4 * 8e-5
    assert (dX.cpu().double() - want[3] @ heads[1].double()).abs().max() < 4 * 8e-5 / n * 0.1 * 16
