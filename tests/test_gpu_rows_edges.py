"""GPU tests of the operators on rows of logits at the edges of their contract:
calls at once, many short rows, rows of every place in memory, the same inputs
through different divisions."""
import math

import pytest

import rows_ref as ref
from test_gpu_distill import blank, inputs as distill_inputs, run
from test_gpu_logprobs import TYPES, check, code, dt, forward, gradient, inputs, put

pytestmark = pytest.mark.gpu


def test_two_calls_at_once(ctx):
    """The operators share nothing but the status word: calls on two streams of one context do not disturb each other."""
    import torch
    streams = [torch.cuda.Stream() for _ in range(2)]
    sides = []
    for seed in range(2):
        x, tokens = inputs(seed, 60, 50257, "f32")
        _, ids, t, w = distill_inputs(seed, 60, 50257, 40, "f32")
        n = x.shape[0]
        f = lambda *s: torch.zeros(*s, device="cuda")  # noqa: E731
        sides.append(dict(x=x, gx=put(x), tokens=tokens, tok=tokens.cuda(), ids=ids, gi=ids.cuda(), t=t, gt=t.cuda(), w=w, gw=w.cuda(),
                          f=[f(n) for _ in range(4)], top=torch.zeros(n, 30, dtype=torch.int32, device="cuda"), lp=f(n, 30),
                          loss=[f(n) for _ in range(3)], dx=f(n, 50257), dy=f(n, 50257), one=torch.ones(n, device="cuda")))
    torch.cuda.synchronize()
    for _ in range(5):
        for s, d in zip(streams, sides):
            ctx.logprobs(d["gx"], d["tok"], *d["f"], d["top"], d["lp"], stream=s)
            ctx.distill(d["gx"], d["gi"], d["gt"], d["loss"][0], d["gw"], d["dx"], d["loss"][1], d["loss"][2], stream=s)
            ctx.logprobs_grad(d["gx"], d["tok"], d["f"][2], d["f"][3], d["dy"], d["one"], d["f"][1], d["one"], stream=s)
    torch.cuda.synchronize()
    for d in sides:
        check(d["f"] + [d["top"], d["lp"]], *ref.logprobs(d["x"], d["tokens"], 1.0, 30))
        check(d["loss"] + [d["dx"]], *ref.distill(d["x"], d["ids"], d["t"], 1.0, d["w"], torch.float32))
        want, tol = ref.logprobs_grad(d["x"], d["tokens"], 1.0, torch.ones(60), torch.ones(60), torch.float32)
        check([d["dy"]], [want], [tol])
    ctx.sync_status()


@pytest.mark.parametrize("V", [1, 3, 40])
def test_many_short_rows(ctx, V):
    """More rows than a grid's y or z dimension holds."""
    import torch
    n = 100003
    x, tokens = inputs(V, n, V, "bf16", left=0.1)
    check(forward(ctx, put(x), tokens, 1.0, min(V, 2)), *ref.logprobs(x, tokens, 1.0, min(V, 2)))
    dl = torch.ones(n)
    want, tol = ref.logprobs_grad(x, tokens, 1.0, dl, dl, torch.float16)
    check([gradient(ctx, put(x), tokens, 1.0, dl, dl, "f16")], [want], [tol])
    ids = torch.randint(-1, V, (n, 3), generator=torch.Generator().manual_seed(1)).to(torch.int32)
    t = torch.randn(n, 3, generator=torch.Generator().manual_seed(2))
    want, tol = ref.distill(x, ids, t, 1.0, None, torch.bfloat16)
    check(run(ctx, put(x), ids, t, 1.0, None, blank(x, "bf16")), want, tol)
    ctx.sync_status()


@pytest.mark.parametrize("dtype", TYPES)
def test_every_place_in_memory(ctx, dtype):
    """Rows and gradients that begin at each place of a 32-byte unit, alike and differently; rows shorter than a unit."""
    import torch
    for V in (5, 33, 700):
        x, tokens = inputs(V, 2, V, dtype)
        _, ids, t, w = distill_inputs(V, 2, V, 4, dtype, empty=0.0)
        dl = torch.tensor([1.0, -0.5])
        lp = ref.logprobs(x, tokens, 1.3, min(V, 5))
        for at in range(17):
            gx = put(x, 1, at)
            check(forward(ctx, gx, tokens, 1.3, min(V, 5)), *lp)
            for d in TYPES:
                for at2 in (at, at + 1, 0):
                    want, tol = ref.logprobs_grad(x, tokens, 1.3, dl, dl, dt(d))
                    out = blank(x, d, 1, at2)
                    check([gradient(ctx, gx, tokens, 1.3, dl, dl, d, out=out)], [want], [tol])
                    want, tol = ref.distill(x, ids, t, 1.3, w, dt(d))
                    other = blank(x, d, 1, at2)
                    check(run(ctx, gx, ids, t, 1.3, w, other), want, tol)
                    for o in (out, other):               # what lies between the rows and behind them stays
                        assert (o.as_strided((1,), (1,), o.storage_offset() + V) == 7.0).all()
                        assert (o.as_strided((8,), (1,), o.storage_offset() + 2 * V + 1) == 7.0).all()
    ctx.sync_status()


@pytest.mark.parametrize("dtype", TYPES)
def test_alternatives_do_not_depend_on_the_batch(ctx, dtype):
    """One row alone (eight blocks), in a small batch and in a large one (one block): the same places, the same logits there."""
    import torch
    V = 90001
    x, tokens = inputs(3, 1, V, dtype)
    x = x.float().round().to(dt(dtype)) if dtype == "f32" else x        # ties in every type
    first = None
    for n in (1, 4, 30, 160):
        got = forward(ctx, put(x.expand(n, V)), tokens.expand(n).contiguous(), 1.0, 200)
        assert (got[4] == got[4][:1]).all() and (got[2] == got[2][0]).all()
        first = first or got
        assert torch.equal(got[4][0], first[4][0])
        assert (got[5][0] - first[5][0]).abs().max() < 2.0 ** -17        # two sums, each within 2^-18
    ctx.sync_status()


def test_sorted_rows_of_many_batches(ctx):
    """The largest logits all in one place, more of them than a block's candidates hold: every group of them is looked through."""
    import torch
    V = 200000
    i = torch.arange(V, dtype=torch.float32)
    rows = torch.stack([i * 1e-4, -i * 1e-4, torch.where(i > V - 5000, 1.0, 0.0), torch.where((i // 16) % 3 == 0, 2.0, 1.0),
                        torch.full((V,), -2.5), torch.where(i < 3000, 3.0 - i * 1e-5, -i)])
    for n in (6, 240):
        x = rows.repeat(n // 6, 1)
        for k in (1, 100, 256):
            got = forward(ctx, put(x), torch.full((n,), 5, dtype=torch.int32), 1.0, k)
            want, tol = ref.logprobs(rows, torch.full((6,), 5, dtype=torch.int32), 1.0, k)
            for at in range(0, n, 6):
                if at in (0, n - 6):
                    check([g[at:at + 6] for g in got], want, tol)
                else:
                    assert torch.equal(got[4][at:at + 6], got[4][:6])
    ctx.sync_status()


def test_loss_of_a_teacher_that_is_the_student(ctx):
    """All of a small vocabulary listed, the teacher's logits the row's own: the loss is 0 and so is the gradient."""
    import torch
    n, V = 20, 200
    x, _ = inputs(1, n, V, "f32")
    ids = torch.stack([torch.randperm(V, generator=torch.Generator().manual_seed(i)) for i in range(n)]).to(torch.int32)
    t = x.gather(1, ids.long())
    got = run(ctx, put(x), ids, t, 1.0, None, blank(x, "f32"))
    # p and q are each within 2^-18 of the same number, and differ from it by no more
    assert got[0].abs().max() < 2.0 ** -17 * 12 and got[3].abs().max() < 2.0 ** -17
    ctx.sync_status()


def test_large_weights_and_temperatures(ctx):
    import torch
    x, ids, t, w = distill_inputs(4, 9, 3001, 12, "f32", empty=0.0)
    for T in (1e-4, 0.01, 100.0, 1e4):
        want, tol = ref.distill(x, ids, t, T, w * 1e6, torch.float32)
        check(run(ctx, put(x), ids, t, T, w * 1e6, blank(x, "f32")), want, tol)
    assert math.isfinite(float(want[0].max()))
    ctx.sync_status()


def test_too_many_rows_are_refused(ctx):
    import tier_b200 as tk
    import torch
    x = torch.zeros(64, device="cuda")
    for n, V in ((2 ** 31 - 1, 1 << 14), (1 << 24, 1 << 23)):
        st = ctx.lib.tk_logprobs(ctx.h, n, V, x.data_ptr(), 0, V, None, 1.0, None, x.data_ptr(), None, None, 0, None, None, None)
        assert st == tk.TK_ERR_INVALID


def test_calls_that_follow_each_other_at_once(ctx):
    """A chain of short calls, each on what the one before left: the next call's blocks come early and wait for it."""
    import torch
    n, V, k = 6, 9001, 16
    x, tokens = inputs(5, n, V, "f32")
    gx, tok = put(x), tokens.cuda()
    f = [torch.zeros(n, device="cuda") for _ in range(4)]
    ids, lp = torch.zeros(n, k, dtype=torch.int32, device="cuda"), torch.zeros(n, k, device="cuda")
    one, loss, buf = torch.ones(n, device="cuda"), torch.zeros(n, device="cuda"), torch.zeros(n, V, device="cuda")
    for turn in range(40):
        ids.fill_(-1)                                     # (what a call that did not wait would see)
        f[2].fill_(1e30)
        ctx.logprobs(gx, tok, *f, ids, lp)
        ctx.distill(gx, ids, lp, loss, one, buf)          # its own ids and values: just written
        ctx.distill(gx, ids, lp, loss)
        ctx.logprobs_grad(gx, tok, f[2], f[3], buf, one, f[1], one)
        ctx.logprobs(buf, None, top_ids=ids, top_logp=lp)  # of the gradient: just written over the other one
        if turn % 13:
            continue
        torch.cuda.synchronize()
        want, tol = ref.logprobs_grad(x, tokens, 1.0, torch.ones(n), torch.ones(n), torch.float32)
        check([buf], [want], [tol])
        top = ref.logprobs(buf.cpu(), None, 1.0, k)
        check([ids, lp], top[0][4:], top[1][4:])
        t = ref.logprobs(x, None, 1.0, k)[0]
        want, tol = ref.distill(x, t[4].to(torch.int32), t[5].float(), 1.0, None, None)
        # (the teacher's values are fp32 log-probabilities, off by 2^-18 and their rounding: q and the loss follow them)
        assert (loss.cpu().double() - want[0]).abs().max() <= tol[0].max() + 2.0 ** -17 * (1 + want[0].max())
    ctx.sync_status()


def test_entries_below_the_least_number_do_not_count(ctx):
    """A q below 2^-126 is 0, though its weight before the division by their sum is above: a row of -inf there has a loss."""
    import torch
    n, V, k = 3, 5000, 256
    x, _ = inputs(2, n, V, "f32")
    ids = torch.arange(k, dtype=torch.int32).repeat(n, 1)
    t = torch.zeros(n, k)
    t[0, 200], t[1, 255], t[2, 7] = -85.0, -87.0, -83.0       # the others' sum is 255: q = 2^-130.6, 2^-133.5 and 2^-127.7
    for r, at in enumerate((200, 255, 7)):
        x[r, at] = -math.inf
    want, tol = ref.distill(x, ids, t, 1.0, None, torch.float32)
    assert want[0].isfinite().all()
    got = run(ctx, put(x), ids, t, 1.0, None, blank(x, "f32"))
    check(got, want, tol)
    check(run(ctx, put(x), ids, t, 1.0, None), want[:3], tol[:3])
    dx = blank(x, "f32")
    ctx.distill_grad(put(x), ids.cuda(), t.cuda(), got[1], got[2], dx)
    check([dx], want[3:], tol[3:])
    for o in (got[3].cpu(), dx.cpu()):
        assert all(o[r, at] == 0 for r, at in enumerate((200, 255, 7)))
    t[:, 100] = -74.0                                         # 2^-114.8: counts
    x[:, 100] = -math.inf
    want, tol = ref.distill(x, ids, t, 1.0, None, torch.float32)
    got = run(ctx, put(x), ids, t, 1.0, None, blank(x, "f32"))
    assert (got[0] == math.inf).all()
    check(got, want, tol)
    ctx.sync_status()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,V", [(300, 40001), (200, 65536)])
def test_gradients_of_many_batches_a_block(ctx, n, V, dtype):
    """Rows enough that a block takes several batches of one, whole ones and a last one that is not: in place, into another
    type's rows on other boundaries (element by element), with and without the entropy."""
    import torch
    x, tokens = inputs(n, n, V, dtype, left=0.1)
    g = torch.Generator().manual_seed(n)
    dl, de = torch.randn(n, generator=g), 0.1 * torch.randn(n, generator=g)
    other = {"f32": "bf16", "f16": "f32", "bf16": "f16"}[dtype]
    for a, b, d, at in ((dl, de, dtype, 0), (dl, de, other, 0), (dl, None, other, 3), (None, de, dtype, 1)):
        want, tol = ref.logprobs_grad(x, tokens, 0.8, a, b, dt(d))
        gx = put(x)
        check([gradient(ctx, gx, tokens, 0.8, a, b, d, out=gx if a is dl and d == dtype else blank(x, d, at, at))], [want], [tol])
    _, ids, t, w = distill_inputs(n, n, V, 40, dtype, twice=0.2)
    for d, at in ((dtype, 0), (other, 0), (other, 3)):
        want, tol = ref.distill(x, ids, t, 1.5, w, dt(d))
        gx = put(x)
        st = run(ctx, gx, ids, t, 1.5, w)
        check(run(ctx, gx, ids, t, 1.5, w, blank(x, d, at, at)), want, tol)
        dx = gx if d == dtype else blank(x, d, at, at)
        ctx.distill_grad(gx, ids.cuda(), t.cuda(), st[1], st[2], dx, w.cuda(), temperature=1.5, x_dtype=code(gx), d_dtype=code(dx))
        check([dx], want[3:], tol[3:])
    ctx.sync_status()


def test_gradients_of_rows_that_hold_no_distribution(ctx):
    """They are reported as the forward pass reports them; where no gradient is asked for, they are zero and are not."""
    import tier_b200 as tk
    import torch
    n, V = 7, 9001
    x, tokens = inputs(7, n, V, "f32")
    x[0, 77], x[2, 8999], x[4] = math.nan, math.inf, -math.inf
    _, ids, t, w = distill_inputs(7, n, V, 10, "f32", empty=0.0, short=0.0)
    gx, tok, one = put(x), tokens.cuda(), torch.ones(n, device="cuda")
    f = [torch.zeros(n, device="cuda") for _ in range(4)]
    ctx.logprobs(gx, tok, *f)
    loss = run(ctx, gx, ids, t, 1.0, None)
    with pytest.raises(tk.TierkError):
        ctx.sync_status()
    none, good = [0, 2, 4], [1, 3, 5, 6]
    calls = [lambda d, g: ctx.logprobs_grad(gx, tok, f[2], f[3], d, g, f[1], None),
             lambda d, g: ctx.logprobs_grad(gx, None, f[2], f[3], d, None, f[1], g),
             lambda d, g: ctx.distill_grad(gx, ids.cuda(), t.cuda(), loss[1], loss[2], d, g)]
    for call in calls:
        dx = blank(x, "f32")
        call(dx, one)
        with pytest.raises(tk.TierkError) as e:
            ctx.sync_status()
        assert e.value.status == tk.TK_ERR_DEVICE
        assert dx[none].isnan().all() and dx[good].isfinite().all()
        some = one.clone()
        some[none] = 0.0
        call(dx, some)
        ctx.sync_status()
        assert (dx[none] == 0).all() and dx[good].isfinite().all()


@pytest.mark.parametrize("T", [1.0, 0.37])
def test_rows_that_rise_slowly(ctx, T):
    """One block a row, whose maximum moves in each of 256 batches by little: no weight decays, and each is scaled again and
    again.  The sums keep the bound of 64 roundings."""
    import torch
    n, batches = 320, 256
    rise = 2.0 ** torch.linspace(-13, 1, n, dtype=torch.float64)
    v = (rise[:, None] * torch.arange(batches, dtype=torch.float64) * T / batches).float()       # by 2^-13 to 2 from end to end
    v[::2] += rise[::2, None].float() * torch.arange(batches) * T                                # and a batch
    x = torch.empty(n, batches, 8192, device="cuda")
    x.copy_(v[:, :, None])
    x = x.view(n, -1)
    y = (v.double() - v.double()[:, -1:]) / T                # sums over the batches, 8192 logits alike in each
    S = 8192 * y.exp().sum(1)
    Y = -(8192 * y.exp() * y).sum(1) / S                     # mean |y|
    e = 2.0 ** -18 + 2.0 ** -22 + 2.0 ** -22 * Y
    logp, ent = y[:, 5] - S.log(), S.log() + Y
    tokens = torch.full((n,), 5 * 8192 + 9, dtype=torch.int32)
    want = [logp, ent, v[:, -1].double(), S]
    tol = [e + 2.0 ** -23 * logp.abs(), (e + 2.0 ** -22) * (2 + 2 * ent + S.log()), torch.zeros(n, dtype=torch.float64), (e + 2.0 ** -24) * S]
    for k in (0, 20):
        got = forward(ctx, x, tokens, T, k)
        check(got[:4], want, tol)
    out = [torch.zeros(n, device="cuda") for _ in range(3)]
    ids, t = tokens[:, None].cuda(), torch.zeros(n, 1, device="cuda")
    dx = torch.empty(n, x.shape[1], dtype=torch.bfloat16, device="cuda")
    for grad in ({}, {"dlogits": dx, "d_dtype": 2}):
        ctx.distill(x, ids, t, out[0], rmax=out[1], rsum=out[2], temperature=T, **grad)
        check(out, [-logp, want[2], S], [e + (2.0 ** -20 + 2.0 ** -24) * logp.abs(), tol[2], tol[3]])
    ctx.sync_status()


def test_the_longest_rows_that_rise_slowly(ctx):
    """1024 batches of one block, their maxima apart by so little that all weigh alike, so that an exponential's error a step
    would add up.  A weight is off by 4 roundings (2^-24 each: its exponential), 7 in its batch, 3 to bring its lanes
    together, in the mean 3.5 as other batches come and 3.5 times 2.5 as the reference moves, and the result by one: 28,
    and the steps' own 2^-22 |y|."""
    import torch
    n, batches = 300, 1024
    x = torch.empty(n, batches, 8192, device="cuda")
    step = 2.0 ** torch.linspace(-22, -9, n, dtype=torch.float64)
    v = (step[:, None] * torch.arange(batches, dtype=torch.float64)).float()
    x.copy_(v[:, :, None])
    x = x.view(n, -1)
    y = v.double() - v.double()[:, -1:]
    S = 8192 * y.exp().sum(1)
    Y = -(8192 * y.exp() * y).sum(1) / S
    e = 28 * 2.0 ** -24 + 2.0 ** -22 * Y
    tokens = torch.zeros(n, dtype=torch.int32)
    for k in (0, 3):
        check(forward(ctx, x, tokens, 1.0, k)[2:4], [v[:, -1].double(), S], [torch.zeros(n, dtype=torch.float64), e * S])
    out = [torch.zeros(n, device="cuda") for _ in range(2)]
    ctx.distill(x, tokens[:, None].cuda(), torch.zeros(n, 1, device="cuda"), rmax=out[0], rsum=out[1])
    check(out, [v[:, -1].double(), S], [torch.zeros(n, dtype=torch.float64), e * S])
    ctx.sync_status()


@pytest.mark.parametrize("dtype", TYPES)
def test_more_candidates_than_fit_beside_the_ends(ctx, dtype):
    """Rows off every boundary, half of whose logits reach the bound: more than a block's candidates hold, with up to 30 ends
    beside them.  Often enough for a slow load of an end to come behind all units' candidates."""
    import torch
    n, V, k = 2000, 3798, 256
    g = torch.Generator(device="cuda").manual_seed(3)
    x = torch.randn(n, V, generator=g, device="cuda") * 2
    x[:, 250:2210] += 5
    x = put(x.to(dt(dtype)), 13, 7)
    order = x.float().sort(dim=1, descending=True, stable=True)
    want = order.indices[:, :k].to(torch.int32)
    ids, lp, wrong = torch.zeros(n, k, dtype=torch.int32, device="cuda"), torch.zeros(n, k, device="cuda"), 0
    for _ in range(200):
        ids.fill_(-1)
        ctx.logprobs(x, top_ids=ids, top_logp=lp, x_dtype=code(x))
        wrong = wrong + (ids != want).any(1).sum()
    assert wrong.item() == 0
    exact = torch.log_softmax(x.double(), 1).gather(1, want.long())
    assert (lp.double() - exact).abs().max() < 2.0 ** -17
    ctx.sync_status()
