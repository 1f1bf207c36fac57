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
