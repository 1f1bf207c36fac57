"""The serving entry points on the host: refusals that need no GPU, and the
binding's structures against the header's."""
import ctypes
import re

from conftest import ROOT


def test_null_contexts_are_refused():
    import tier_b200 as tk
    from tier_b200 import build
    build.build()
    lib = tk.load()
    c, s = tk.KvCache(), tk.Seqs()
    p, q = ctypes.byref(c), ctypes.byref(s)
    for st in (lib.tk_kv_append(None, p, q, None, None, 0, 0, 0, None), lib.tk_kv_read(None, p, q, None, None, 0, 0, 0, None),
               lib.tk_kv_attend(None, p, q, None, 0, 0, 4, 1.0, 0, None, 0, None),
               lib.tk_draft_verify(None, 1, None, 1, 10, None, 10, None, 0, None, None, None, 1.0, None, None, None, None)):
        assert st == tk.TK_ERR_INVALID and b"null context" in lib.tk_last_error_string()


def test_structures_match_the_header():
    import tier_b200 as tk
    text = (ROOT / "include" / "tierk.h").read_text()
    for name, cls in (("tk_kvcache", tk.KvCache), ("tk_seqs", tk.Seqs)):
        body = re.search(r"typedef struct %s \{(.*?)\} %s;" % (name, name), text, re.S).group(1)
        fields = []
        for decl in body.split(";"):
            m = re.match(r"\s*(?:const\s+)?(int32_t|int|void)\s+(.*)", decl.strip(), re.S)
            if m:
                fields += [(f.strip().lstrip("*"), "*" in f) for f in m.group(2).split(",")]
        assert [f for f, _ in fields] == [f for f, _ in cls._fields_]
        assert [ctypes.c_void_p if ptr else ctypes.c_int for _, ptr in fields] == [t for _, t in cls._fields_]


def test_references_agree_with_themselves():
    """Packing and unpacking invert each other, and every value n * d is exact in fp16."""
    import numpy as np
    import kv_ref as ref
    rng = np.random.default_rng(0)
    x = (rng.standard_normal((50, 2, 128)) * np.exp(rng.uniform(-8, 8, (50, 2, 1)))).astype(np.float32)
    n, d = ref.quantize(x)
    back = ref.unpack(ref.pack(n), d)
    assert np.array_equal(back, n * np.repeat(d.astype(np.float64), 32, -1))
    assert np.array_equal(back, back.astype(np.float16).astype(np.float64))
    step = np.repeat(np.abs(x.reshape(50, 2, 4, 32)).max(-1) / 8, 32, -1)
    assert (np.abs(back - x) <= step * (1 + 2.0 ** -5)).all()


def test_tensors_that_do_not_hold_the_rows_are_refused():
    """The library cannot see an address's memory end: the bindings refuse other types, too few rows and other devices
    before it is called.  (No context here: what passes them ends in the library's refusal of a null one.)"""
    import pytest
    import tier_b200 as tk
    import torch
    ctx = tk.Context.__new__(tk.Context)
    ctx.lib, ctx.h, ctx.device = tk.load(), None, -1       # device -1: the tensors' own here
    cache, seqs = tk.KvCache(8, 16, 2, 64), tk.Seqs(1, 5, 5, 1)

    def refused(what, fn, *args, **kw):
        with pytest.raises(tk.TierkError) as e:
            fn(*args, stream=0, **kw)
        assert e.value.status == tk.TK_ERR_INVALID and what in str(e.value), str(e.value)

    x, wide = torch.zeros(5, 128), torch.zeros(5, 256)
    for fn in (ctx.kv_append, ctx.kv_read):
        name = "tk_" + fn.__name__
        for k, v in ((x, x), (torch.zeros(7, 136)[:, :128], x), (x.view(5, 2, 64), x), (x.view(torch.int32), x)):
            refused(name + ": null context", fn, cache, seqs, k, v)
        refused(name + ": null context", fn, cache, seqs, x.flatten(), x, ldk=128)
        refused(name + ": null context", fn, cache, seqs, x.half(), x.half(), tk.DT_F16)
        refused(name + ": k holds torch.float16", fn, cache, seqs, x.half(), x)
        refused(name + ": v holds torch.bfloat16", fn, cache, seqs, x.half(), x.bfloat16(), tk.DT_F16)
        refused(name + ": k holds torch.float32", fn, cache, seqs, x, x, tk.DT_BF16)
        refused(name + ": v holds no 5 rows", fn, cache, seqs, x, x[:4])
        refused(name + ": v holds no 5 rows", fn, cache, seqs, x, x[:0])
        refused(name + ": k holds no 5 rows", fn, cache, seqs, wide, x, ldk=300)
        refused(name + ": k holds no 5 rows", fn, cache, seqs, wide[:, 136:], x)
        refused(name + ": v has rows that are not contiguous", fn, cache, seqs, x, torch.zeros(128, 5).t(), ldv=128)
    refused("tk_kv_attend: null context", ctx.kv_attend, cache, seqs, wide, 4, wide)
    refused("tk_kv_attend: q holds no 5 rows", ctx.kv_attend, cache, seqs, x.view(5, 128), 4, wide, ldq=256)
    refused("tk_kv_attend: out holds no 5 rows", ctx.kv_attend, cache, seqs, wide, 4, wide[:4])
    refused("tk_kv_attend: out holds torch.float64", ctx.kv_attend, cache, seqs, wide, 4, wide.double())
    ctx.device = 0
    refused("tk_kv_attend: q is not on device 0", ctx.kv_attend, cache, seqs, wide, 4, wide)
    cache._device = 1
    refused("tk_kv_attend: cache and batch must be on device 0", ctx.kv_attend, cache, seqs, wide, 4, wide)
    ctx.device = -1

    i = lambda n: torch.zeros(n, dtype=torch.int32)  # noqa: E731
    f = torch.zeros
    good = dict(target=f(5, 100), tokens=i(5), row_start=i(3), u_accept=f(5), u_sample=f(2), n_accept=i(2), next_token=i(2),
                logp=f(5), draft=f(5, 100))
    for kw in ({}, {"draft": None}, {"logp": None}, {"temperature": 0.0, "u_accept": None, "u_sample": None}, {"u_accept": f(4)},
               {"target": f(5, 120)[:, :100]}):
        refused("tk_draft_verify: null context", ctx.draft_verify, **{**good, **kw})
    for name, bad in (("target", f(5, 100).double()), ("draft", f(4, 100)), ("draft", f(5, 120)[:, :99]),
                      ("draft", f(5, 100).half()), ("tokens", i(4)), ("tokens", i(5).long()), ("tokens", i(10)[::2]),
                      ("row_start", i(2)), ("u_accept", f(3)), ("u_accept", f(5).double()), ("u_sample", f(1)), ("next_token", i(1)),
                      ("next_token", i(2).long()), ("logp", f(4)), ("logp", f(5).half())):
        refused("tk_draft_verify: " + name, ctx.draft_verify, **{**good, name: bad})
    with pytest.raises(ValueError):
        tk.make_seqs(i(2), i(1), i(3).view(1, 3), 1, 1)
    with pytest.raises(ValueError):
        tk.alloc_kvcache(2, 16, 1, 64, device="cpu")
