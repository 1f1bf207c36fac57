"""GPU parity of the 4-bit key/value cache (tk_kv_append, tk_kv_read) and the
attention over it (tk_kv_attend).

The cache's bytes must equal the plain rule's, and read back exactly.
Attention is held, value by value, to
    |out - exact| <= u * |exact| + e * sum_j p_j |v_j|
u: the output type's half unit (2^-24, 2^-11, 2^-8).  e for fp16 and bf16 rows:
2^-11 (the probabilities' one rounding to fp16) + 2e-5; for fp32 rows 2e-5: the
scores here stay below 40, q's two fp16 parts leave 2^-22 of each, the fp32
sums of 128 terms about as much again, so a probability is off by at most
40 * 2^-22 * 2 = 1.9e-5 of itself.
"""
import numpy as np
import pytest

import kv_ref as ref

pytestmark = pytest.mark.gpu
DTYPES = ["f32", "f16", "bf16"]


def types(name):
    import torch
    import tier_b200 as tk
    return {"f32": (torch.float32, tk.DT_F32, 2.0 ** -24), "f16": (torch.float16, tk.DT_F16, 2.0 ** -11),
            "bf16": (torch.bfloat16, tk.DT_BF16, 2.0 ** -8)}[name]


def dev(a):
    import torch
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def device_cache(cache):
    import tier_b200 as tk
    return tk.make_kvcache(*(dev(cache[x]) for x in ("k_q", "k_s", "v_q", "v_s")))


def device_seqs(q_start, kv_len, pages, max_new=None):
    import tier_b200 as tk
    n = int(q_start[-1])
    return tk.make_seqs(dev(q_start), dev(kv_len), dev(pages), n,
                        int(np.diff(q_start).max()) if max_new is None else max_new)


def run_attend(ctx, cache, bat, q, heads, dtype, window=0, scale=None, pad=0, out_fill=7.0, stream=None):
    """q float64-able [tokens, heads * dim] -> out float64, through rows `pad` elements wider than they need."""
    import torch
    tt, dt, _ = types(dtype)
    qd = torch.full((q.shape[0], q.shape[1] + pad), 3.0, dtype=tt, device="cuda")
    qd[:, : q.shape[1]] = dev(q).to(tt)
    out = torch.full_like(qd, out_fill)
    torch.cuda.synchronize()
    kc = device_cache(cache) if isinstance(cache, dict) else cache
    ctx.kv_attend(kc, device_seqs(*bat[:3]), qd, heads, out, x_dtype=dt, window=window, scale=scale, stream=stream)
    ctx.sync_status(stream)
    assert (out[:, q.shape[1]:] == out_fill).all()        # nothing outside the rows
    return qd[:, : q.shape[1]].double().cpu().numpy(), out[:, : q.shape[1]].double().cpu().numpy()


def check_attend(out, exact, reach, dtype):
    u = types(dtype)[2]
    e = 2e-5 if dtype == "f32" else 2.0 ** -11 + 2e-5
    bad = np.abs(out - exact) > u * np.abs(exact) + e * reach + 1e-30
    assert not bad.any(), (bad.sum(), float(np.abs(out - exact).max()), np.argwhere(bad)[:3].tolist())


def attend_case(ctx, new, kv, heads, kv_heads, dim, page, dtype, window=0, seed=0, pad=0, garbage=True):
    rng = np.random.default_rng(seed)
    bat = ref.batch(rng, new, kv, page)
    cache = ref.random_cache(rng, bat[3], page, kv_heads, dim)
    if garbage:   # rows that no sequence holds: infinities and NaN
        held = np.zeros((bat[3], page), bool)
        for b, c in enumerate(kv):
            for t in range(c):
                held[bat[2][b, t // page], t % page] = True
        g = ref.random_cache(rng, bat[3], page, kv_heads, dim, garbage=True)
        for x in ("k_s", "v_s"):
            cache[x] = np.where(held[:, None, :, None], cache[x], g[x])
    q = rng.standard_normal((int(bat[0][-1]), heads * dim)) * 2
    qr, out = run_attend(ctx, cache, bat, q, heads, dtype, window, pad=pad)
    exact, reach = ref.attend(cache, bat[0], bat[1], bat[2], qr, heads, kv_heads, dim, dim ** -0.5, window)
    check_attend(out.reshape(exact.shape), exact, reach, dtype)


# ---- append and read back ------------------------------------------------------
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim,heads,page,new,kv", [
    (128, 8, 64, [1], [1]), (128, 2, 16, [5, 0, 33], [20, 7, 33]), (64, 3, 32, [1, 1, 1, 64], [1, 100, 33, 64]),
    (64, 1, 256, [7, 250], [7, 300]), (128, 1, 128, [129], [1000])])
def test_append_writes_the_rules_bytes(ctx, dtype, dim, heads, page, new, kv):
    import torch
    rng = np.random.default_rng(dim + sum(new))
    q_start, kv_len, pages, total = ref.batch(rng, new, kv, page)
    tt, dt, _ = types(dtype)
    cache = ref.random_cache(rng, total, page, heads, dim)
    n, w = sum(new), heads * dim
    x = {}
    for s in "kv":
        a = rng.standard_normal((n, heads, dim // 32, 32)) * np.exp(rng.uniform(-4, 4, (n, heads, dim // 32, 1)))
        a[rng.random(a.shape[:3]) < 0.1] = 0                      # groups of zeros
        a[rng.random(a.shape[:3]) < 0.1] *= 2.0 ** -24            # below fp16's normal numbers
        a[rng.random(a.shape[:3]) < 0.05] *= 1e6 / 8              # beyond the scales' range
        a[0, 0, 0, :] = np.where(np.arange(32) % 2, -1.5, 1.5)    # several of the largest magnitude
        x[s] = torch.zeros(n, w + 16, dtype=tt, device="cuda")
        if dtype == "f16":
            a = np.clip(a, -65504, 65504)
        x[s][:, :w] = dev(a.reshape(n, w)).to(tt)
    kc = device_cache(cache)
    sq = device_seqs(q_start, kv_len, pages)
    ctx.kv_append(kc, sq, x["k"], x["v"], x_dtype=dt)
    ctx.sync_status()
    got = dict(zip(("k_q", "k_s", "v_q", "v_s"), (t.cpu().numpy() for t in kc._owner)))
    for s in "kv":
        m, d = ref.quantize(x[s][:, :w].float().cpu().numpy().reshape(n, heads, dim))
        for b in range(len(new)):
            for i in range(new[b]):
                t, r = kv[b] - new[b] + i, int(q_start[b]) + i
                cache[s + "_q"][pages[b, t // page], :, t % page] = ref.pack(m[r])
                cache[s + "_s"][pages[b, t // page], :, t % page] = d[r]
    for name, a in got.items():
        assert np.array_equal(a.view(np.uint8), cache[name].view(np.uint8)), name
    # read back, exactly, in every type that holds the values
    for out in ("f32", "f16"):
        to, do, _ = types(out)
        k, v = (torch.full((n, w + 8), 5.0, dtype=to, device="cuda") for _ in "kv")
        ctx.kv_read(kc, sq, k, v, out_dtype=do)
        ctx.sync_status()
        for s, r in (("k", k), ("v", v)):
            m, d = ref.quantize(x[s][:, :w].float().cpu().numpy().reshape(n, heads, dim))
            want = (m * np.repeat(d.astype(np.float64), 32, -1)).reshape(n, w)
            assert np.array_equal(r[:, :w].double().cpu().numpy(), want)
            assert (r[:, w:] == 5).all()


def test_append_rounds_to_within_half_a_step(ctx):
    """|x - n d| <= |d| / 2, but for the side of the range that 4 bits lack (up to 1 step) and d's own rounding."""
    import torch
    import tier_b200 as tk
    rng = np.random.default_rng(5)
    q_start, kv_len, pages, total = ref.batch(rng, [200], [200], 64)
    kc = tk.alloc_kvcache(total, 64, 4, 128)
    x = dev(rng.standard_normal((200, 512)).astype(np.float32))
    k, v = torch.empty_like(x), torch.empty_like(x)
    sq = device_seqs(q_start, kv_len, pages)
    ctx.kv_append(kc, sq, x, -x)
    ctx.kv_read(kc, sq, k, v)
    ctx.sync_status()
    for a, r in ((x, k), (-x, v)):
        step = a.view(200, 16, 32).abs().amax(-1, keepdim=True) / 8
        err = (a - r).view(200, 16, 32).abs()
        assert bool((err <= step * (1 + 2.0 ** -5)).all())
        assert float((err <= step * (0.5 + 2.0 ** -5)).float().mean()) > 0.95


def test_append_reports_values_that_are_not_finite(ctx):
    import torch
    import tier_b200 as tk
    rng = np.random.default_rng(6)
    q_start, kv_len, pages, total = ref.batch(rng, [3], [3], 16)
    kc = tk.alloc_kvcache(total, 16, 1, 64)
    k = torch.ones(3, 64, device="cuda")
    k[1, 5], k[1, 40], k[2, 0] = float("nan"), float("inf"), float("-inf")
    sq = device_seqs(q_start, kv_len, pages)
    ctx.kv_append(kc, sq, k, torch.ones_like(k))
    with pytest.raises(tk.TierkError) as e:
        ctx.sync_status()
    assert e.value.status == tk.TK_ERR_DEVICE
    r = torch.empty_like(k)
    ctx.kv_read(kc, sq, r, torch.empty_like(k))
    ctx.sync_status()
    want = torch.where(torch.isfinite(k), k, torch.zeros_like(k))
    assert torch.equal(r, want)


def test_rows_before_the_cache_and_empty_batches(ctx):
    """More new tokens than cached ones: the early rows are not appended, read back as zeros and attend to nothing."""
    import torch
    import tier_b200 as tk
    rng = np.random.default_rng(7)
    q_start, kv_len, pages = np.array([0, 5, 9], np.int32), np.array([2, 0], np.int32), np.zeros((2, 1), np.int32)
    kc = tk.alloc_kvcache(2, 16, 2, 64)
    sq = device_seqs(q_start, kv_len, pages)
    x = dev(rng.standard_normal((9, 128)).astype(np.float32))
    ctx.kv_append(kc, sq, x, x)
    r, s = torch.full_like(x, 9.0), torch.full_like(x, 9.0)
    ctx.kv_read(kc, sq, r, s)
    out = torch.full((9, 256), 9.0, device="cuda")
    ctx.kv_attend(kc, sq, torch.randn(9, 256, device="cuda"), 4, out)
    ctx.sync_status()
    assert (r[:3] == 0).all() and (r[5:] == 0).all() and (r[3:5] != 0).any()
    assert (out[:3] == 0).all() and (out[5:] == 0).all() and (out[3:5] != 0).any()
    rows = kc._owner[1][0]                       # page 0's key scales: two tokens and nothing behind them
    assert bool((rows[:, :2] != 0).all()) and bool((rows[:, 2:] == 0).all())
    # no sequences, no tokens, no new tokens: nothing to do, and no pointer is looked at
    for empty in ((0, 0, 0), (2, 0, 3), (2, 4, 0)):
        z = tk.Seqs(empty[0], empty[1], empty[2], 1, None, None, None)
        ctx.kv_attend(kc, z, x, 4, out, ldq=256, ldo=256)
        ctx.kv_append(kc, z, x, x)
        ctx.kv_read(kc, z, x, x)
    ctx.sync_status()


# ---- attention -----------------------------------------------------------------
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim,heads,kv_heads", [(128, 4, 1), (128, 8, 8), (64, 6, 2), (64, 16, 2), (128, 12, 1)])
def test_attend_single_tokens(ctx, dtype, dim, heads, kv_heads):
    """One new token a sequence: lengths around every tile edge, an empty sequence, ones without new tokens."""
    kv = [1, 2, 31, 32, 33, 64, 65, 127, 129, 0, 300, 17]
    attend_case(ctx, [1] * 11 + [0], kv, heads, kv_heads, dim, 16, dtype, seed=dim + heads)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("page", [16, 32, 64, 128, 256])
def test_attend_pages(ctx, dtype, page):
    attend_case(ctx, [1, 3, 2], [page - 1, 2 * page + 1, 517], 4, 2, 64, page, dtype, seed=page)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("new,heads,kv_heads", [(2, 8, 2), (5, 8, 2), (8, 8, 1), (3, 4, 4), (16, 8, 2), (9, 9, 3)])
def test_attend_drafted_tokens(ctx, dtype, new, heads, kv_heads):
    attend_case(ctx, [new, 1, new - 1, new], [new, 40, 333, 1100], heads, kv_heads, 128, 64, dtype, seed=new)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim,new,kv", [(128, [130], [130]), (64, [257, 1, 64], [257, 300, 100]), (128, [33, 300], [600, 301]),
                                        (64, [100, 0, 129], [1000, 5, 129])])
def test_attend_prompts(ctx, dtype, dim, new, kv):
    attend_case(ctx, new, kv, 8, 2, dim, 32, dtype, seed=dim + new[0])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("window", [1, 5, 64, 100, 1000])
@pytest.mark.parametrize("new,kv", [([1, 1, 1], [3, 200, 1000]), ([4, 7], [150, 700]), ([200, 140], [200, 500])])
def test_attend_windows(ctx, dtype, window, new, kv):
    attend_case(ctx, new, kv, 4, 2, 64, 16, dtype, window=window, seed=window)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("new,heads", [(1, 4), (4, 8), (70, 2)])
def test_attend_strided_rows_and_long_context(ctx, dtype, new, heads):
    """Rows wider than their heads; a context long enough to be divided among many thread blocks."""
    attend_case(ctx, [new], [9000], heads, 2, 128 if new == 1 else 64, 64, dtype, seed=new, pad=24)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("new,heads,kv_heads", [(1, 24, 1), (3, 8, 1), (7, 8, 2), (8, 4, 1), (1, 31, 1)])
def test_attend_all_row_counts_of_the_streaming_kernel(ctx, dtype, new, heads, kv_heads):
    """17 to 32 rows per key/value head."""
    attend_case(ctx, [new, max(1, new - 1), new], [2000, 33, new], heads, kv_heads, 128 if new == 3 else 64, 64, dtype, seed=heads)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("new", [1, 9])
def test_attend_many_sequences_of_different_length(ctx, dtype, new):
    """More sequences than a warp has lanes, and more heads than thread blocks: a few long, most short, some empty."""
    rng = np.random.default_rng(21)
    kv = [int(x) for x in rng.integers(new, 60, 70)]
    for b in range(0, 70, 9):
        kv[b] = 1500 + b
    news = [0 if b % 13 == 5 else new for b in range(70)]
    attend_case(ctx, news, kv, 16 if new == 9 else 8, 8 if new == 1 else 2, 64, 16, dtype, seed=22)


def test_append_many_sequences(ctx):
    """More than 32 and more than 1024 sequences: the places of their tokens."""
    import torch
    import tier_b200 as tk
    for B in (33, 1100):
        rng = np.random.default_rng(B)
        new = [int(x) for x in rng.integers(0, 3, B)]
        kv = [n + int(x) for n, x in zip(new, rng.integers(0, 20, B))]
        q_start, kv_len, pages, total = ref.batch(rng, new, kv, 16)
        kc = tk.alloc_kvcache(total, 16, 1, 64)
        sq = device_seqs(q_start, kv_len, pages)
        x = rng.standard_normal((sum(new), 64)).astype(np.float32)
        ctx.kv_append(kc, sq, dev(x), dev(-x))
        ctx.sync_status()
        k_q, v_q = kc._owner[0].cpu().numpy(), kc._owner[2].cpu().numpy()
        m, _ = ref.quantize(x)
        w, _ = ref.quantize(-x)
        for b in range(B):
            for i in range(new[b]):
                t, r = kv[b] - new[b] + i, int(q_start[b]) + i
                assert np.array_equal(k_q[pages[b, t // 16], 0, t % 16], ref.pack(m[r]))
                assert np.array_equal(v_q[pages[b, t // 16], 0, t % 16], ref.pack(w[r]))


@pytest.mark.parametrize("dtype", DTYPES)
def test_attend_a_value_far_above_the_rest(ctx, dtype):
    """Scores that climb along the context and one key far above all others, each way round."""
    rng = np.random.default_rng(11)
    for where in (0, 500, 999):
        bat = ref.batch(rng, [2, 40], [1000, 1000], 64)
        cache = ref.random_cache(rng, bat[3], 64, 1, 64)
        for b in range(2):
            for t in range(1000):
                cache["k_s"][bat[2][b, t // 64], :, t % 64] = np.float16(0.0625) if t != where else np.float16(0.5)
                cache["k_q"][bat[2][b, t // 64], :, t % 64] = ref.pack(np.full((1, 64), 1 + t // 250, np.int8))
        q = np.abs(rng.standard_normal((42, 4 * 64))) * 0.5 + 0.25
        qr, out = run_attend(ctx, cache, bat, q, 4, dtype)
        exact, reach = ref.attend(cache, bat[0], bat[1], bat[2], qr, 4, 1, 64, 0.125, 0)
        check_attend(out.reshape(exact.shape), exact, reach, dtype)


@pytest.mark.parametrize("dtype", DTYPES)
def test_attend_wide_ranges(ctx, dtype):
    """Values near the cache's limits and far below them, and an all-zero query (every key alike)."""
    rng = np.random.default_rng(12)
    bat = ref.batch(rng, [1, 3, 30], [50, 60, 70], 16)
    for scale in (2.0 ** -20, 2.0 ** 11):
        cache = ref.random_cache(rng, bat[3], 16, 2, 64)
        cache["v_s"] = (np.sign(cache["v_s"]) * scale).astype(np.float16)
        q = rng.standard_normal((34, 4 * 64))
        q[::3] = 0
        qr, out = run_attend(ctx, cache, bat, q, 4, dtype)
        exact, reach = ref.attend(cache, bat[0], bat[1], bat[2], qr, 4, 2, 64, 0.125, 0)
        u, e = types(dtype)[2], 2e-5 if dtype == "f32" else 2.0 ** -11 + 2e-5
        small = 2.0 ** -25 if dtype == "f16" else 0.0     # fp16 results below its normal numbers
        assert (np.abs(out.reshape(exact.shape) - exact) <= u * np.abs(exact) + e * reach + small).all()


def test_attend_query_that_is_not_finite_stays_in_its_row(ctx):
    rng = np.random.default_rng(13)
    for new in (1, 6, 64):
        bat = ref.batch(rng, [new, new], [100, 90], 16)
        cache = ref.random_cache(rng, bat[3], 16, 2, 64)
        q = rng.standard_normal((2 * new, 4 * 64))
        _, good = run_attend(ctx, cache, bat, q, 4, "f32")
        q[0, 64:128] = np.nan
        q[new, 70] = np.inf
        _, out = run_attend(ctx, cache, bat, q, 4, "f32")
        same = np.ones_like(good, bool)
        same[0, 64:128] = same[new, 64:128] = False
        assert np.array_equal(out[same], good[same])
        assert np.isnan(out[0, 64:128]).all() and np.isnan(out[new, 64:128]).all()


@pytest.mark.parametrize("dtype", DTYPES)
def test_attend_scale_and_repeatability(ctx, dtype):
    """Another scale (zero and negative ones too); the same call twice gives the same bits, and on another stream."""
    import torch
    rng = np.random.default_rng(14)
    bat = ref.batch(rng, [1, 4, 50], [3000, 500, 64], 32)
    cache = ref.random_cache(rng, bat[3], 32, 2, 128)
    q = rng.standard_normal((55, 8 * 128))
    for scale in (0.0, -0.05, 0.2):
        qr, out = run_attend(ctx, cache, bat, q, 8, dtype, scale=scale)
        exact, reach = ref.attend(cache, bat[0], bat[1], bat[2], qr, 8, 2, 128, np.float32(scale), 0)
        check_attend(out.reshape(exact.shape), exact, reach, dtype)
        _, again = run_attend(ctx, cache, bat, q, 8, dtype, scale=scale)
        _, other = run_attend(ctx, cache, bat, q, 8, dtype, scale=scale, stream=torch.cuda.Stream())
        assert np.array_equal(out, again) and np.array_equal(out, other)


def test_attend_pages_beyond_32_bit_offsets(ctx):
    """A cache whose last pages lie more than 2^32 bytes from its start."""
    import torch
    import tier_b200 as tk
    heads, page, dim = 64, 256, 128
    n_pages = 2 ** 32 // (heads * page * dim // 2) + 3
    q = [torch.empty(n_pages, heads, page, dim // 2, dtype=torch.uint8, device="cuda") for _ in "kv"]
    s = [torch.empty(n_pages, heads, page, dim // 32, dtype=torch.float16, device="cuda") for _ in "kv"]
    kc = tk.make_kvcache(q[0], s[0], q[1], s[1])
    rng = np.random.default_rng(15)
    for new in (1, 20):
        q_start, kv_len, pages = np.array([0, 300], np.int32), np.array([300], np.int32), np.array([[n_pages - 1, n_pages - 2]], np.int32)
        x = [dev(rng.standard_normal((300, heads * dim)).astype(np.float32)) for _ in "kv"]
        ctx.kv_append(kc, device_seqs(q_start, kv_len, pages), x[0], x[1])
        bat = (np.array([0, new], np.int32), kv_len, pages)
        qq = rng.standard_normal((new, heads * dim))
        qr, out = run_attend(ctx, kc, bat, qq, heads, "f32")
        small = {n: t[n_pages - 2:].cpu().numpy() for n, t in zip(("k_q", "k_s", "v_q", "v_s"), kc._owner)}
        exact, reach = ref.attend(small, bat[0], kv_len, np.array([[1, 0]], np.int32), qr, heads, heads, dim, dim ** -0.5, 0)
        check_attend(out.reshape(exact.shape), exact, reach, "f32")


def test_batches_that_do_not_fit_are_reported(ctx):
    """Contents of the device arrays that do not fit raise the status; the other sequences' results stand."""
    import torch
    import tier_b200 as tk
    rng = np.random.default_rng(16)
    for new in (1, 40):
        good = ref.batch(rng, [new, new], [70, 80], 16)
        cache = ref.random_cache(rng, good[3], 16, 2, 64)
        q = rng.standard_normal((2 * new, 4 * 64))
        _, want = run_attend(ctx, cache, good, q, 4, "f32")
        kc = device_cache(cache)
        qd = dev(q.astype(np.float32))

        def broken(**kw):
            a = dict(q_start=good[0].copy(), kv_len=good[1].copy(), pages=good[2].copy(), max_new=new)
            a.update(kw)
            out = torch.zeros_like(qd)
            ctx.kv_attend(kc, device_seqs(a["q_start"], a["kv_len"], a["pages"], a["max_new"]), qd, 4, out)
            with pytest.raises(tk.TierkError) as e:
                ctx.sync_status()
            assert e.value.status == tk.TK_ERR_DEVICE
            return out.double().cpu().numpy()

        pages = good[2].copy()
        pages[0, 1] = good[3]
        assert np.array_equal(broken(pages=pages)[new:], want[new:])
        pages[0, 1] = -1
        assert np.array_equal(broken(pages=pages)[new:], want[new:])
        assert np.array_equal(broken(kv_len=np.array([pages.shape[1] * 16 + 1, 80], np.int32))[new:], want[new:])
        assert np.array_equal(broken(kv_len=np.array([-1, 80], np.int32))[new:], want[new:])
        # q_start that goes back, and beyond the rows (n_tokens stays the last entry: 2 * new)
        broken(q_start=np.array([new + 1, new, 2 * new], np.int32))
        broken(q_start=np.array([-1, new, 2 * new], np.int32))


def test_attend_in_a_captured_graph(ctx):
    """Captured once, replayed after the batch's numbers changed on the device."""
    import torch
    import tier_b200 as tk
    rng = np.random.default_rng(17)
    q_start, kv_len, pages, total = ref.batch(rng, [2, 2], [200, 100], 32)
    cache = ref.random_cache(rng, total, 32, 2, 128)
    kc = device_cache(cache)
    sq = device_seqs(q_start, kv_len, pages)
    q = dev(rng.standard_normal((4, 8 * 128)).astype(np.float32))
    out = torch.zeros_like(q)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    ctx.kv_attend(kc, sq, q, 8, out, stream=side)          # grows the workspace before the capture
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=side):
        ctx.kv_attend(kc, sq, q, 8, out, stream=side)
    for lens in ([200, 100], [57, 2], [33, 100]):
        sq._owner[1].copy_(torch.tensor(lens, dtype=torch.int32))
        out.zero_()
        g.replay()
        torch.cuda.synchronize()
        exact, reach = ref.attend(cache, q_start, np.array(lens), pages, q.double().cpu().numpy(), 8, 2, 128, 128 ** -0.5, 0)
        check_attend(out.double().cpu().numpy().reshape(exact.shape), exact, reach, "f32")
    ctx.sync_status()


def test_drafted_decoding_example(ctx):
    """The example's greedy text is the same with drafts and without (each step's tokens through all operators)."""
    import importlib.util
    from conftest import ROOT
    spec = importlib.util.spec_from_file_location("draft_decode", ROOT / "examples" / "draft_decode.py")
    ex = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(ex)
    prompts = [[3, 14, 15, 92, 65, 3, 14], [2, 71, 82, 2, 71], [1] * 40]
    plain, _, _ = ex.generate(ex.Decoder(ctx), prompts, 24, drafts=0)
    texts, taken, offered = ex.generate(ex.Decoder(ctx), prompts, 24, drafts=4)
    for a, b in zip(plain, texts):
        n = min(len(a), len(b))
        assert a[:n] == b[:n]
    assert 0 <= taken <= offered and offered > 0
    warm, _, _ = ex.generate(ex.Decoder(ctx), prompts, 4, drafts=4, temperature=1.0, seed=5)
    assert all(0 <= t < 1000 for w in warm for t in w)


def test_refusals(ctx):
    import torch
    import tier_b200 as tk
    x = torch.zeros(4, 256, device="cuda")
    seqs = device_seqs(np.array([0, 4], np.int32), np.array([4], np.int32), np.zeros((1, 1), np.int32))
    good = tk.alloc_kvcache(2, 16, 2, 64)

    def refused(status, fn):
        with pytest.raises(tk.TierkError) as e:
            fn()
        assert e.value.status == status and "tk_kv_" in str(e.value)

    def attend(c=good, s=seqs, q=x, heads=4, out=x, **kw):
        return lambda: ctx.kv_attend(c, s, q, heads, out, **kw)

    def cache(**kw):
        c = tk.KvCache(*(kw.get(n, getattr(good, n)) for n, _ in tk.KvCache._fields_))
        c._owner = good._owner
        return c

    def batch(**kw):
        b = tk.Seqs(*(kw.get(n, getattr(seqs, n)) for n, _ in tk.Seqs._fields_))
        b._owner = seqs._owner
        return b

    refused(tk.TK_ERR_UNSUPPORTED, attend(cache(head_dim=96)))
    for c in (cache(page_tokens=8), cache(page_tokens=48), cache(page_tokens=512), cache(n_pages=0), cache(n_kv_heads=0),
              cache(k_q=None), cache(v_s=None), cache(k_s=good.k_s + 2), cache(v_q=good.v_q + 8)):
        refused(tk.TK_ERR_INVALID, attend(c))
        refused(tk.TK_ERR_INVALID, lambda: ctx.kv_append(c, seqs, x, x))
        refused(tk.TK_ERR_INVALID, lambda: ctx.kv_read(c, seqs, x, x))
    for s in (batch(n_seqs=-1), batch(n_tokens=-1), batch(max_new=-1), batch(max_pages=0), batch(max_pages=1 << 28),
              batch(q_start=None), batch(kv_len=None), batch(pages=None)):
        refused(tk.TK_ERR_INVALID, attend(s=s))
        refused(tk.TK_ERR_INVALID, lambda: ctx.kv_append(good, s, x, x))
    refused(tk.TK_ERR_INVALID, attend(heads=3))
    refused(tk.TK_ERR_INVALID, attend(heads=0))
    refused(tk.TK_ERR_INVALID, attend(window=-1))
    refused(tk.TK_ERR_INVALID, attend(scale=float("nan")))
    refused(tk.TK_ERR_INVALID, attend(scale=float("inf")))
    refused(tk.TK_ERR_INVALID, attend(x_dtype=7))
    refused(tk.TK_ERR_INVALID, attend(ldq=255))
    refused(tk.TK_ERR_INVALID, attend(ldo=258))
    refused(tk.TK_ERR_INVALID, attend(q=x[:, 1:], ldq=256))
    refused(tk.TK_ERR_INVALID, attend(out=x[:, 2:], ldo=256))
    refused(tk.TK_ERR_INVALID, lambda: ctx.kv_append(good, seqs, x, x, ldk=64))
    refused(tk.TK_ERR_INVALID, lambda: ctx.kv_append(good, seqs, x[:, 1:], x))
    with pytest.raises(ValueError):
        tk.make_kvcache(*(t[:, :1] for t in good._owner))
    with pytest.raises(ValueError):
        tk.make_seqs(seqs._owner[0].long(), seqs._owner[1], seqs._owner[2], 4, 4)
    ctx.sync_status()


@pytest.mark.parametrize("rising", [False, True])
@pytest.mark.parametrize("dtype,dim,new,seqs", [
    ("f32", 128, 40, 90), ("f32", 64, 40, 90), ("f16", 128, 100, 90), ("f16", 64, 30, 150),   # row sets
    ("f32", 128, 1, 330), ("f32", 64, 7, 330), ("f16", 128, 2, 330), ("bf16", 128, 1, 330),     # streamed
])
def test_attend_long_sums(ctx, dtype, dim, new, seqs, rising):
    """One block or warp adds 20000 keys' values, all of one sign, in sequences enough that none is cut into short parts.

    A sum that lost 2^-24 of itself with each of its 16-key products would be 7e-5 to 1.5e-4 off; what is allowed is 2e-5 of
    sum p |v| (and the rounding of 16-bit outputs and weights), of which 128 such losses take 0.8e-5, 512 3.1e-5.
    `rising`: scores grow by 2^60 along the keys, so that the reference moves in the midst of sums.
    """
    kv, page, heads = 20000, 256, 4
    need = -(-kv // page)
    rng = np.random.default_rng(11)
    cache = ref.random_cache(rng, need, page, 1, dim)
    cache["v_q"] = rng.integers(1, 8, cache["v_q"].shape, dtype=np.uint8) * 16 + rng.integers(1, 8, cache["v_q"].shape, dtype=np.uint8)
    cache["v_s"] = np.abs(cache["v_s"]) + np.float16(2.0 ** -6)
    cache["v_s"] = ref.round_bits(cache["v_s"].astype(np.float64), 8).astype(np.float16)
    q = rng.standard_normal((new, heads * dim)) * 0.3
    if rising:
        cache["k_q"] = cache["k_q"] & 0x77                                  # 0 to 7
        at = (np.arange(need * page).reshape(need, 1, page, 1) + 1) / (need * page)
        cache["k_s"] = ref.round_bits(np.broadcast_to(0.1 * at, cache["k_s"].shape), 8).astype(np.float16)
        q = np.abs(q) * 60 * np.log(2) * np.sqrt(dim) / (0.1 * 3.5 * np.abs(q).reshape(new, heads, dim).sum(-1).repeat(dim, -1))
    pages = np.tile(np.arange(need, dtype=np.int32), (seqs, 1))
    bat = (np.arange(seqs + 1, dtype=np.int32) * new, np.full(seqs, kv, np.int32), pages, need)
    qr, out = run_attend(ctx, cache, bat, np.tile(q, (seqs, 1)), heads, dtype)
    exact, reach = ref.attend(cache, bat[0][:2], bat[1][:1], pages[:1], qr[:new], heads, 1, dim, dim ** -0.5, 0)
    check_attend(out.reshape(seqs, *exact.shape), exact[None], reach[None], dtype)
