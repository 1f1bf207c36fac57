"""GPU tests of the verification of drafted tokens at the edges of its contract."""
import numpy as np
import pytest

from test_gpu_verify import run

pytestmark = pytest.mark.gpu


def test_draws_of_the_largest_vocabulary(ctx):
    """2^23 tokens, rows off a 16-byte boundary and sequences enough for one block each: a warp's longest sums.

    2^19 + 1 tokens are alike and the others impossible: a token's weight, floor(2^38 / (2^19 + 1)) = 2^19 - 1, fills the
    low half of the sums, so the draw is known: floor(goal / (2^19 - 1)).
    """
    import torch
    V, B, some = 1 << 23, 100, (1 << 19) + 1
    flat = torch.full((B * V + 1,), -float("inf"), device="cuda")
    target = flat[1:].view(B, V)
    target[:, :some] = 0.25
    us = ((np.arange(B) + 0.5) / B).astype(np.float32)
    acc, nxt = (torch.full((B,), -7, dtype=torch.int32, device="cuda") for _ in range(2))
    start = torch.arange(B + 1, dtype=torch.int32, device="cuda")
    ctx.draft_verify(target, torch.zeros(B, dtype=torch.int32, device="cuda"), start, torch.zeros(B, device="cuda"),
                     torch.from_numpy(us).cuda(), acc, nxt)
    ctx.sync_status()
    weight = (1 << 38) // some
    assert weight == (1 << 19) - 1
    want = [(weight * some * int(u * np.float32(2 ** 24)) >> 24) // weight for u in us]
    assert (acc == 0).all() and nxt.tolist() == want


def test_rows_behind_a_refusal_may_hold_anything(ctx):
    """Nothing of the rows after the refused one is needed, nor a sequence's last row of draft logits."""
    V = 5000
    rng = np.random.default_rng(61)
    base = rng.standard_normal((5, V)).astype(np.float32)
    start, tokens = np.array([0, 3, 5], np.int32), np.zeros(5, np.int32)
    tokens[1:] = base.argmax(1)[:-1]
    tokens[1] = base[0].argmin()
    us = np.full(2, 0.5, np.float32)
    for with_draft in (False, True):
        t, d = base.copy(), base.copy()
        d[0, tokens[1]] = 20.0                            # drafted far above its probability: refused
        t[1:3] = np.nan
        d[1:3] = np.nan
        d[4] = np.nan
        ua = np.array([0.999, 0.999, 0.999, 0.0, 0.999], np.float32)
        acc, nxt, logp = run(ctx, start, t, d if with_draft else None, tokens, ua, us, 1.0)
        ctx.sync_status()
        assert acc.tolist() == [0, 1] and (nxt >= 0).all() and nxt[0] != tokens[1]
        assert (logp[1:3] == 0).all() and np.isfinite(logp).all()
