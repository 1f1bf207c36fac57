"""The operators on rows of logits on the host: refusals that need no GPU, and
the plain forms that the GPU tests compare with, against each other."""
import math

import pytest
import torch

import rows_ref as ref


def test_null_contexts_are_refused():
    import tier_b200 as tk
    from tier_b200 import build
    build.build()
    lib = tk.load()
    for st in (lib.tk_logprobs(None, 1, 10, None, 0, 10, None, 1.0, None, None, None, None, 0, None, None, None),
               lib.tk_logprobs_grad(None, 1, 10, None, 0, 10, None, 1.0, None, None, None, None, None, None, 0, 10, None),
               lib.tk_distill(None, 1, 10, None, 0, 10, 1, None, None, 1.0, None, None, None, None, None, 0, 10, None),
               lib.tk_distill_grad(None, 1, 10, None, 0, 10, 1, None, None, 1.0, None, None, None, None, 0, 10, None)):
        assert st == tk.TK_ERR_INVALID and b"null context" in lib.tk_last_error_string()


def test_tensors_that_do_not_hold_the_rows_are_refused():
    """As for the serving bindings: other types, too few rows and other devices, before the library is called."""
    import tier_b200 as tk
    ctx = tk.Context.__new__(tk.Context)
    ctx.lib, ctx.h, ctx.device = tk.load(), None, -1       # device -1: the tensors' own here
    i = lambda *n: torch.zeros(*n, dtype=torch.int32)  # noqa: E731
    f = torch.zeros

    def refused(what, fn, **kw):
        with pytest.raises(tk.TierkError) as e:
            fn(stream=0, **kw)
        assert e.value.status == tk.TK_ERR_INVALID and what in str(e.value), str(e.value)

    good = {ctx.logprobs: dict(logits=f(5, 100), tokens=i(5), logp=f(5), entropy=f(5), rmax=f(5), rsum=f(5), top_ids=i(5, 3),
                               top_logp=f(5, 3)),
            ctx.logprobs_grad: dict(logits=f(5, 100), tokens=i(5), rmax=f(5), rsum=f(5), dlogits=f(5, 100), d_logp=f(5),
                                    entropy=f(5), d_entropy=f(5)),
            ctx.distill: dict(logits=f(5, 100), ids=i(5, 3), teacher=f(5, 3), loss=f(5), weight=f(5), dlogits=f(5, 100),
                              rmax=f(5), rsum=f(5)),
            ctx.distill_grad: dict(logits=f(5, 100), ids=i(5, 3), teacher=f(5, 3), rmax=f(5), rsum=f(5), dlogits=f(5, 100),
                                   weight=f(5))}
    for fn, kw in good.items():
        name = "tk_" + fn.__name__
        for some in ({}, {"logits": f(5, 120)[:, :100]}):
            refused(name + ": null context", fn, **{**kw, **some})
        refused(name + ": logits holds torch.float64", fn, **{**kw, "logits": f(5, 100).double()})
        refused(name + ": logits has rows that are not contiguous", fn, **{**kw, "logits": f(5, 200)[:, ::2]})
        for key in set(kw) - {"logits", "dlogits", "ids", "top_ids"}:
            refused(f"{name}: {key} must be", fn, **{**kw, key: kw[key][:-1]})
            refused(f"{name}: {key} must be", fn, **{**kw, key: kw[key].double()})
        for key in {"ids", "top_ids"} & set(kw):
            refused(f"{name}: {key} must be a matrix of 5 rows", fn, **{**kw, key: i(15)})
            refused(f"{name}: {key} must be a matrix of 5 rows", fn, **{**kw, key: i(4, 3)})
            refused(f"{name}: {key} must be 15 contiguous int32", fn, **{**kw, key: i(5, 4)[:, :3]})
            refused(f"{name}: {key} must be 15 contiguous int32", fn, **{**kw, key: i(5, 3).long()})
        if "dlogits" in kw:
            refused(name + ": dlogits holds no 5 rows", fn, **{**kw, "dlogits": f(4, 100)})
            refused(name + ": dlogits holds torch.float16", fn, **{**kw, "dlogits": f(5, 100).half()})
            refused(name + ": null context", fn, **{**kw, "dlogits": f(5, 100).half()}, d_dtype=tk.DT_F16)
        ctx.device = 0
        refused(name + ": logits is not on device 0", fn, **kw)
        ctx.device = -1


def test_what_belongs_to_the_places_has_their_shape():
    """A teacher's values, or the buffer for the alternatives', wider than the places or turned: their numbers would be
    taken for other rows'."""
    import tier_b200 as tk
    ctx = tk.Context.__new__(tk.Context)
    ctx.lib, ctx.h, ctx.device = tk.load(), None, -1
    x, v, ids = torch.zeros(5, 100), torch.zeros(5), torch.zeros(5, 3, dtype=torch.int32)
    calls = {"top_logp": [lambda t: ctx.logprobs(x, top_ids=ids, top_logp=t, stream=0)],
             "teacher": [lambda t: ctx.distill(x, ids, t, v, stream=0), lambda t: ctx.distill_grad(x, ids, t, v, v, x.clone(), stream=0)]}
    for name, fns in calls.items():
        for fn in fns:
            for shape in ((5, 6), (3, 5), (6, 3), (15,), (5, 3, 1), (5, 2), (1, 5, 3)):
                with pytest.raises(tk.TierkError) as e:
                    fn(torch.zeros(shape))
                assert e.value.status == tk.TK_ERR_INVALID and f"{name} must be a matrix of" in str(e.value), str(e.value)
            with pytest.raises(tk.TierkError, match="null context"):
                fn(torch.zeros(5, 3))


def test_a_refused_launch_leaves_no_error_behind(tmp_path):
    """The next call would launch, and return the old error as its own."""
    import subprocess
    from pathlib import Path
    from tier_b200 import build
    if not Path(build.NVCC).exists():
        pytest.skip("nvcc not available")
    objs = [build.BUILD / (s.stem + ".o") for s in build.sources()]
    build.build(force=not all(o.exists() and o.stat().st_mtime >= s.stat().st_mtime for o, s in zip(objs, build.sources())))
    src, exe = Path(__file__).parent / "refused_launch.cu", tmp_path / "refused_launch"
    r = subprocess.run([build.NVCC, *build.ARCH, "-std=c++17", "-I", str(build.PKG.parent / "include"), "-I", str(build.CSRC), str(src),
                        *map(str, objs), "-o", str(exe), "-ldl", "-lpthread", "-lrt",
                        *(f"-Xlinker=--wrap={f}" for f in ("cudaLaunchKernelExC", "cudaGetLastError", "cudaFuncSetAttribute"))],
                       capture_output=True, text=True, timeout=600)
    assert r.returncode == 0, r.stdout + r.stderr
    r = subprocess.run([str(exe)], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0 and "0 failures" in r.stdout, r.stdout + r.stderr


def test_plain_forms_agree_with_automatic_gradients():
    g = torch.Generator().manual_seed(0)
    x = torch.randn(6, 40, generator=g, dtype=torch.float64) * 2
    x[3, 5:9] = -math.inf
    tokens, T = torch.tensor([0, 5, -1, 7, 39, 2], dtype=torch.int32), 1.4
    a, b = torch.randn(6, generator=g), torch.randn(6, generator=g)
    z = x.clone().requires_grad_()
    lp = torch.log_softmax(z / T, 1)
    p = lp.exp()
    ent = -torch.where(p > 0, p * torch.where(p > 0, lp, torch.zeros_like(lp)), torch.zeros_like(p)).sum(1)
    live = tokens >= 0
    logp = lp.gather(1, tokens.clamp(min=0).long()[:, None])[:, 0]
    tokens[3] = 20
    logp = lp.gather(1, tokens.clamp(min=0).long()[:, None])[:, 0]
    (want,) = torch.autograd.grad((live * (a.double() * logp + b.double() * ent)).sum(), z)
    got, _ = ref.logprobs_grad(x, tokens, T, a, b, torch.float32)
    assert torch.allclose(got, want.nan_to_num(0.0), atol=1e-12)
    val, _ = ref.logprobs(x, tokens, T, 3)
    assert torch.allclose(val[1], torch.where(live, ent, torch.zeros_like(ent)).detach())
    ids = torch.randint(40, (6, 7), generator=g).to(torch.int32)
    ids[1, 3:], ids[2], ids[4, 1] = -1, -1, ids[4, 0]
    x[3, 5:9] = 0.0
    t, w, z = torch.randn(6, 7, generator=g), torch.rand(6, generator=g), x.clone().requires_grad_()
    q, live = ref.teacher(ids, t, 40, T)
    lp = torch.log_softmax(z / T, 1).gather(1, ids.clamp(min=0).long())
    loss = torch.where(q > 0, q * (torch.where(q > 0, q, torch.ones_like(q)).log() - lp), torch.zeros_like(q)).sum(1)
    (want,) = torch.autograd.grad((live * w.double() * loss).sum(), z)
    val, _ = ref.distill(x, ids, t, T, w, torch.float32)
    assert torch.allclose(val[3], want, atol=1e-12) and torch.allclose(val[0], torch.where(live, loss, 0.0).detach(), atol=1e-6)
    assert (val[3][2] == 0).all() and not live[2]
