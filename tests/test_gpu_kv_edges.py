"""GPU tests of the 4-bit cache and the attention over it at the edges of their
contract: captured graphs and what is allocated after them, windows of any
size, page ids that do not fit, small weights of fp32 rows, scores near the
limits of fp32, long appends.
Tolerances as in test_gpu_kv.py."""
import numpy as np
import pytest

import kv_ref as ref
import test_gpu_kv
from test_gpu_kv import DTYPES, dev, device_cache, device_seqs, run_attend

pytestmark = pytest.mark.gpu


def check_attend(out, exact, reach, dtype):
    assert np.isfinite(out).all()                          # (a NaN is above no bound)
    test_gpu_kv.check_attend(out, exact, reach, dtype)


class Replayed:
    """Two sequences' drafted rows, long enough to be divided among blocks and joined, captured in a graph."""

    def __init__(self, ctx):
        import torch
        rng = np.random.default_rng(31)
        self.ctx, self.bat = ctx, ref.batch(rng, [2, 2], [3000, 1700], 32)
        self.cache = ref.random_cache(rng, self.bat[3], 32, 2, 128)
        self.q = dev(rng.standard_normal((4, 8 * 128)).astype(np.float32))
        self.out = torch.zeros_like(self.q)
        self.kc, self.sq = device_cache(self.cache), device_seqs(*self.bat[:3])
        self.side = torch.cuda.Stream()
        torch.cuda.synchronize()
        self.call()                                        # sizes the workspace before the capture
        torch.cuda.synchronize()
        self.graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(self.graph, stream=self.side):
            self.call()

    def call(self):
        self.ctx.kv_attend(self.kc, self.sq, self.q, 8, self.out, stream=self.side)

    def check(self):
        import torch
        for _ in range(2):
            self.out.zero_()
            self.graph.replay()
            torch.cuda.synchronize()
            exact, reach = ref.attend(self.cache, *self.bat[:3], self.q.double().cpu().numpy(), 8, 2, 128, 128 ** -0.5, 0)
            check_attend(self.out.double().cpu().numpy().reshape(exact.shape), exact, reach, "f32")
        self.ctx.sync_status()


def larger_calls(ctx):
    """A prompt of many row sets, and decoding of more sequences than the graph's."""
    import torch
    import tier_b200 as tk
    kc = tk.alloc_kvcache(128, 64, 8, 128)
    pages = torch.arange(128, dtype=torch.int32, device="cuda").view(1, -1)
    starts = torch.tensor([0, 8192], dtype=torch.int32, device="cuda")
    q = torch.randn(8192, 32 * 128, device="cuda").bfloat16()
    ctx.kv_attend(kc, tk.make_seqs(starts, starts[1:].clone(), pages, 8192, 8192), q, 32, torch.empty_like(q), x_dtype=tk.DT_BF16)
    n = 300
    sq = tk.make_seqs(torch.arange(n + 1, dtype=torch.int32, device="cuda"), torch.full((n,), 200, dtype=torch.int32, device="cuda"),
                      pages.repeat(n, 1), n, 1)
    ctx.kv_attend(kc, sq, q[:n], 32, torch.empty_like(q[:n]), x_dtype=tk.DT_BF16)
    ctx.sync_status()


def test_replay_after_larger_calls_with_the_workspace_reserved():
    """tk_reserve covers all that a call needs: nothing that a captured graph uses moves afterwards."""
    import tier_b200 as tk
    ctx = tk.Context(0)
    ctx.reserve(256 << 20)
    r = Replayed(ctx)
    r.check()
    size = ctx.lib.tk_workspace_bytes(ctx.h)
    larger_calls(ctx)
    assert ctx.lib.tk_workspace_bytes(ctx.h) == size
    r.check()
    ctx.close()


def test_replay_after_the_workspace_has_grown():
    """A graph captured before a larger call still computes in memory of its own context."""
    import tier_b200 as tk
    ctx = tk.Context(0)
    r = Replayed(ctx)
    size = ctx.lib.tk_workspace_bytes(ctx.h)
    larger_calls(ctx)
    assert ctx.lib.tk_workspace_bytes(ctx.h) > size
    r.check()
    ctx.close()


def test_growth_inside_a_capture_is_refused():
    import torch
    import tier_b200 as tk
    ctx = tk.Context(0)
    side = torch.cuda.Stream()
    kc = tk.alloc_kvcache(2, 16, 1, 64)
    sq = device_seqs(np.array([0, 1], np.int32), np.array([20], np.int32), np.array([[0, 1]], np.int32))
    q = torch.randn(1, 4 * 64, device="cuda")
    out = torch.empty_like(q)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=side):
        with pytest.raises(tk.TierkError) as e:
            ctx.kv_attend(kc, sq, q, 4, out, stream=side)
        out.fill_(3.0)                                     # the capture goes on
    assert e.value.status == tk.TK_ERR_INVALID and "capture" in str(e.value)
    g.replay()
    torch.cuda.synchronize()
    assert (out == 3).all()
    ctx.kv_attend(kc, sq, q, 4, out)
    ctx.sync_status()
    assert (out != 3).any()
    ctx.close()


# ---- windows ---------------------------------------------------------------------
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("new,kv", [([8, 5, 1], [2, 1, 40]), ([64, 200, 40], [2, 50, 90])])
@pytest.mark.parametrize("window", [2 ** 30 - 1, 2 ** 30, 2 ** 31 - 4, 2 ** 31 - 1])
def test_windows_as_large_as_an_int(ctx, dtype, new, kv, window):
    """More new tokens than cached ones, so that rows have negative positions: a window that hides nothing is no window."""
    rng = np.random.default_rng(41)
    bat = ref.batch(rng, new, kv, 16)
    cache = ref.random_cache(rng, bat[3], 16, 2, 64)
    q = rng.standard_normal((sum(new), 4 * 64)) * 2
    qr, none = run_attend(ctx, cache, bat, q, 4, dtype)
    _, out = run_attend(ctx, cache, bat, q, 4, dtype, window=window)
    exact, reach = ref.attend(cache, *bat[:3], qr, 4, 2, 64, 0.125, 0)
    check_attend(out.reshape(exact.shape), exact, reach, dtype)
    assert np.array_equal(out, none)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("new,kv", [([8, 5, 1], [2, 1, 40]), ([64, 200, 40], [2, 50, 90])])
@pytest.mark.parametrize("window", [1, 7, 50])
def test_windows_with_rows_before_the_cache(ctx, dtype, new, kv, window):
    rng = np.random.default_rng(42)
    bat = ref.batch(rng, new, kv, 16)
    cache = ref.random_cache(rng, bat[3], 16, 2, 64)
    q = rng.standard_normal((sum(new), 4 * 64)) * 2
    qr, out = run_attend(ctx, cache, bat, q, 4, dtype, window=window)
    exact, reach = ref.attend(cache, *bat[:3], qr, 4, 2, 64, 0.125, window)
    check_attend(out.reshape(exact.shape), exact, reach, dtype)


# ---- pages -------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("many", [False, True])
def test_append_to_a_page_outside_the_cache_is_skipped(ctx, dtype, many):
    """Its tokens are reported, written nowhere and read back as zeros; every other byte of the cache is as it should be."""
    import torch
    import tier_b200 as tk
    heads, dim, page = (8, 128, 16) if many else (2, 64, 16)
    new = [1300, 40, 30] if many else [20, 40, 30]
    kv = [n + 5 for n in new]
    rng = np.random.default_rng(51)
    q_start, kv_len, pages, total = ref.batch(rng, new, kv, page)
    at0 = np.argwhere(pages[0] == 0)
    if at0.size == 0:                                     # page 0 is some sequence's: here the first one's second page
        pages[pages == 0], pages[0, 1] = pages[0, 1], 0
    pages[1, 1], pages[2, 0] = total, -1
    cache = ref.random_cache(rng, total, page, heads, dim)
    tt, dt = {"f32": (torch.float32, tk.DT_F32), "f16": (torch.float16, tk.DT_F16), "bf16": (torch.bfloat16, tk.DT_BF16)}[dtype]
    x = [dev(rng.standard_normal((sum(new), heads * dim)).astype(np.float32)).to(tt) for _ in "kv"]
    kc, sq = device_cache(cache), device_seqs(q_start, kv_len, pages)
    ctx.kv_append(kc, sq, *x, x_dtype=dt)
    with pytest.raises(tk.TierkError) as e:
        ctx.sync_status()
    assert e.value.status == tk.TK_ERR_DEVICE
    got = dict(zip(("k_q", "k_s", "v_q", "v_s"), (t.cpu().numpy() for t in kc._owner)))
    want = []
    for s, rows in zip("kv", x):
        m, d = ref.quantize(rows.float().cpu().numpy().reshape(-1, heads, dim))
        back = (m * np.repeat(d.astype(np.float64), 32, -1)).reshape(len(m), -1)
        for b in range(3):
            for i in range(new[b]):
                t, r = kv[b] - new[b] + i, int(q_start[b]) + i
                p = pages[b, t // page]
                if not 0 <= p < total:
                    back[r] = 0
                    continue
                cache[s + "_q"][p, :, t % page] = ref.pack(m[r])
                cache[s + "_s"][p, :, t % page] = d[r]
        want.append(back)
    for name, a in got.items():
        assert np.array_equal(a.view(np.uint8), cache[name].view(np.uint8)), name
    out = [torch.full((sum(new), heads * dim), 5.0, device="cuda") for _ in "kv"]
    ctx.kv_read(kc, sq, *out)
    with pytest.raises(tk.TierkError):
        ctx.sync_status()
    for a, w in zip(out, want):
        assert np.array_equal(a.double().cpu().numpy(), w)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("page", [16, 32, 64])
@pytest.mark.parametrize("new", [1, 5, 70])
def test_pages_behind_a_window_are_not_looked_up(ctx, dtype, page, new):
    """Entries of pages that no row sees may be anything: a caller frees those before the window."""
    rng = np.random.default_rng(52)
    kv = [400, 333, 96, 70 + new, 511]
    for window in (1, 17, 40, 100):
        bat = ref.batch(rng, [new] * 5, kv, page)
        cache = ref.random_cache(rng, bat[3], page, 2, 64)
        q = rng.standard_normal((5 * new, 4 * 64)) * 2
        q_start, kv_len, pages = (a.copy() for a in bat[:3])
        for b, c in enumerate(kv):
            pages[b, : max(0, c - new - window + 1) // page] = -1
            pages[b, -(-c // page):] = bat[3] + 7
        qr, out = run_attend(ctx, cache, (q_start, kv_len, pages), q, 4, dtype, window=window)
        exact, reach = ref.attend(cache, *bat[:3], qr, 4, 2, 64, 0.125, window)
        check_attend(out.reshape(exact.shape), exact, reach, dtype)


# ---- fp32 rows -----------------------------------------------------------------------
@pytest.mark.parametrize("where", [0, 700, 1999])
@pytest.mark.parametrize("new,seqs", [(1, 1), (1, 330), (4, 330), (6, 330), (8, 330), (60, 1), (300, 1)])
def test_fp32_rows_whose_mass_lies_on_a_key_of_no_value(ctx, new, seqs, where):
    """One key weighs 2^5 to 2^22 times any other and its value is zero: the others' weights, alike and small, are the
    whole output.  Their two fp16 parts end at 2^-25, the largest weight is 2^14 or more: 2^-17 of a weight that is 2^-22
    of it, within the 2e-5 of every fp32 row.  (330 sequences: none is cut into short parts.)"""
    rng = np.random.default_rng(53)
    kv, page, dim, heads = 2000 + new, 64, 64, 4
    bat = ref.batch(rng, [new], [kv], page)
    cache = ref.random_cache(rng, bat[3], page, 1, dim)
    cache["k_q"][:] = 0
    cache["k_s"][:] = 0.0625
    cache["v_q"] = rng.integers(1, 8, cache["v_q"].shape, dtype=np.uint8) * 17
    cache["v_s"] = np.abs(cache["v_s"]) + np.float16(2.0 ** -6)
    cache["v_s"] = ref.round_bits(cache["v_s"].astype(np.float64), 8).astype(np.float16)
    p, r = bat[2][0, where // page], where % page
    cache["k_q"][p, :, r] = ref.pack(np.full((1, dim), 7, np.int8))
    cache["v_q"][p, :, r] = 0
    gap = rng.uniform(5, 22, (new, heads))                 # of the weights' exponents
    gap[0] = [21.9, 20.3, 18.6, 21.2]
    q = np.repeat(gap * np.log(2) / (0.125 * dim * 7 * 0.0625), dim, -1)
    many = (np.arange(seqs + 1, dtype=np.int32) * new, np.full(seqs, kv, np.int32), np.tile(bat[2], (seqs, 1)), bat[3])
    qr, out = run_attend(ctx, cache, many, np.tile(q, (seqs, 1)), heads, "f32")
    exact, reach = ref.attend(cache, *bat[:3], qr[:new], heads, 1, dim, 0.125, 0)
    check_attend(out.reshape(seqs, *exact.shape), exact[None], reach[None], "f32")


# ---- append and read back of many tokens ----------------------------------------------
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim,heads,page,n", [(128, 8, 64, 1500), (64, 3, 16, 7001), (128, 5, 128, 2200), (64, 17, 256, 1300)])
def test_append_and_read_of_many_tokens(ctx, dtype, dim, heads, page, n):
    """Calls long enough that a warp takes 128 groups of eight of a row; rows whose last warp is not full; every type."""
    import torch
    import tier_b200 as tk
    assert n * heads * dim // 8 > 32 * 32 * 148
    rng = np.random.default_rng(dim + heads)
    new = [n // 3, 0, 1, n - n // 3 - 1]
    kv = [new[0] + 9, 5, 1, new[3]]
    q_start, kv_len, pages, total = ref.batch(rng, new, kv, page)
    tt = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
    dt = {"f32": tk.DT_F32, "f16": tk.DT_F16, "bf16": tk.DT_BF16}
    cache, w, x = ref.random_cache(rng, total, page, heads, dim), heads * dim, {}
    for s in "kv":
        a = rng.standard_normal((n, heads, dim // 32, 32)) * np.exp(rng.uniform(-4, 4, (n, heads, dim // 32, 1)))
        a[rng.random(a.shape[:3]) < 0.05] = 0
        a[rng.random(a.shape[:3]) < 0.05] *= 2.0 ** -24
        a[rng.random(a.shape[:3]) < 0.02] *= 1e6 / 8
        a[:: 97, 0, 0, :] = np.where(np.arange(32) % 2, -1.5, 1.5)
        x[s] = torch.zeros(n, w + 8, dtype=tt[dtype], device="cuda")
        x[s][:, :w] = dev(np.clip(a, -65504, 65504).reshape(n, w)).to(tt[dtype])
    kc, sq = device_cache(cache), device_seqs(q_start, kv_len, pages)
    ctx.kv_append(kc, sq, x["k"], x["v"], x_dtype=dt[dtype])
    ctx.sync_status()
    got = dict(zip(("k_q", "k_s", "v_q", "v_s"), (t.cpu().numpy() for t in kc._owner)))
    seq = np.repeat(np.arange(4), new)
    t = kv_len[seq] - (q_start[seq + 1] - np.arange(n))
    place = (pages[seq, t // page], slice(None), t % page)
    want = {}
    for s in "kv":
        m, d = ref.quantize(x[s][:, :w].float().cpu().numpy().reshape(n, heads, dim))
        cache[s + "_q"][place], cache[s + "_s"][place] = ref.pack(m), d
        want[s] = (m * np.repeat(d.astype(np.float64), 32, -1)).reshape(n, w)
    for name, a in got.items():
        assert np.array_equal(a.view(np.uint8), cache[name].view(np.uint8)), name
    for out in DTYPES:
        k, v = (torch.full((n, w + 8), 5.0, dtype=tt[out], device="cuda") for _ in "kv")
        ctx.kv_read(kc, sq, k, v, out_dtype=dt[out])
        ctx.sync_status()
        for s, r in (("k", k), ("v", v)):
            assert torch.equal(r[:, :w].cpu(), torch.from_numpy(want[s]).to(tt[out])), (s, out)
            assert (r[:, w:] == 5).all()


def test_read_back_in_bf16(ctx):
    """Few tokens; a value n * d of 11 bits is rounded to bf16's 8, ties to even."""
    import torch
    import tier_b200 as tk
    rng = np.random.default_rng(54)
    new, kv = [3, 1, 40], [10, 1, 60]
    q_start, kv_len, pages, total = ref.batch(rng, new, kv, 16)
    cache = ref.random_cache(rng, total, 16, 3, 64)
    kc, sq = device_cache(cache), device_seqs(q_start, kv_len, pages)
    k, v = (torch.full((44, 3 * 64 + 8), 5.0, dtype=torch.bfloat16, device="cuda") for _ in "kv")
    ctx.kv_read(kc, sq, k, v, out_dtype=tk.DT_BF16)
    ctx.sync_status()
    for s, r in (("k", k), ("v", v)):
        values = ref.unpack(cache[s + "_q"], cache[s + "_s"])
        for b in range(3):
            for i in range(new[b]):
                t = kv[b] - new[b] + i
                want = torch.from_numpy(values[pages[b, t // 16], :, t % 16].reshape(-1)).to(torch.bfloat16)
                assert torch.equal(r[q_start[b] + i, :192].cpu(), want)
        assert (r[:, 192:] == 5).all()


def test_scales_whose_power_of_two_overflows_are_refused(ctx):
    """Scores are scale * log2(e) * q . k: such a scale made every score infinite or NaN."""
    import torch
    import tier_b200 as tk
    kc = tk.alloc_kvcache(1, 16, 1, 64)
    sq = device_seqs(np.array([0, 2], np.int32), np.array([9], np.int32), np.zeros((1, 1), np.int32))
    q = torch.zeros(2, 64, device="cuda")
    for scale in (2.5e38, -3.4e38, float("inf")):
        with pytest.raises(tk.TierkError) as e:
            ctx.kv_attend(kc, sq, q, 1, torch.empty_like(q), scale=scale)
        assert e.value.status == tk.TK_ERR_INVALID
    out = torch.full_like(q, 3.0)
    ctx.kv_attend(kc, sq, q, 1, out, scale=2.3e38)
    ctx.sync_status()
    assert (out == 0).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("where", [0, 700, 1999])
@pytest.mark.parametrize("new,seqs", [(1, 1), (4, 100), (8, 100), (60, 1), (300, 1)])
def test_scores_so_large_that_their_rounding_is_whole_powers(ctx, dtype, new, seqs, where):
    """Scores of 2^10 to 2^26.9 in powers of two, whose fp32 steps reach 8: weights stay finite, and the key that leads by
    half a score or more is the output (its weight's one or two fp16 parts over their sum: the tolerance of every row)."""
    rng = np.random.default_rng(55)
    kv, page, dim, heads = 2000 + new, 64, 64, 4
    bat = ref.batch(rng, [new], [kv], page)
    cache = ref.random_cache(rng, bat[3], page, 1, dim)
    cache["k_q"] = ref.pack(rng.integers(-8, 4, (*cache["k_q"].shape[:3], dim)).astype(np.int8))
    cache["k_s"][:] = 500.0
    p, r = bat[2][0, where // page], where % page
    cache["k_q"][p, :, r] = ref.pack(np.full((1, dim), 7, np.int8))
    size = 2.0 ** rng.uniform(10, 26.9, (new, heads))
    size[0] = 2.0 ** np.array([26.9, 25.7, 24.8, 20.6])
    q = np.repeat(size * np.log(2) / (0.125 * dim * 7 * 500.0), dim, -1)
    many = (np.arange(seqs + 1, dtype=np.int32) * new, np.full(seqs, kv, np.int32), np.tile(bat[2], (seqs, 1)), bat[3])
    qr, out = run_attend(ctx, cache, many, np.tile(q, (seqs, 1)), heads, dtype)
    exact, reach = ref.attend(cache, *bat[:3], qr[:new], heads, 1, dim, 0.125, 0)
    check_attend(out.reshape(seqs, *exact.shape), exact[None], reach[None], dtype)
