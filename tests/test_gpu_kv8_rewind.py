"""kv_rewind_q8 with the operators it serves: two sequences, a prompt, drafts and chains
of rewinds.  After each rewind the cache reads as before it, and the next append leaves
the codes of the blocks below its length as they were."""
from __future__ import annotations

import pytest
import torch

from tests.kv8_util import BLOCK, D, DTYPES, EPS, THETA, expected_read, loaded, proj_rows, random_kv

pytestmark = pytest.mark.gpu

B, HQ, HKV, SMAX = 2, 4, 2, 448


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,drafts,lengths", [
    (128, 10, [128, 74]),          # rejected drafts in the slots of the block before the one before
    (128, 10, [128, 128, 64]),
    (330, 16, [330, 320, 256, 200, 74, 5]),
    (330, 0, [266, 202, 138, 74, 10]),
    (384, 16, [384, 256, 129, 128, 127]),
    (448, 0, [448, 384, 191, 80, 64, 0]),
    (200, 5, [185, 150, 143]),
])
def test_chains_of_rewinds(device, dtype, n, drafts, lengths):
    import dflash_mlx as dm

    k, v = random_kv(B, HKV, n, seed=n)
    cache, lens = loaded(device, k, v, [n] * B, SMAX, dtype)
    w = torch.ones(D, dtype=torch.bfloat16, device=device)

    def append(T, length):
        rows = proj_rows(B, T, HQ, HKV, seed=length).to(device)
        at = torch.full((B,), length, dtype=torch.int32, device=device)
        dm.attn_prep_q8(rows, w, w, at, cache, num_heads=HQ, rot_dims=32, rope_base=THETA, eps=EPS)

    if drafts:
        append(drafts, n)
    written = n + drafts
    for L in lengths:
        written = dm.kv_rewind_q8(cache, L, written)
        assert written >= L
        at = torch.full((B,), L, dtype=torch.int32, device=device)
        whole = L // BLOCK * BLOCK
        for x, got in zip((k, v), dm.kv_read_q8(cache, at, L)):
            for b in range(B):
                codes = expected_read(x[b], n, 0, L, dtype)  # every complete block of the history from its codes
                y = got[b].cpu()
                assert torch.equal(y[:, :whole], codes[:, :whole]), L
                # the open block: the history's bf16, or what its code stands for where the slots were taken
                a, c = x[b, :, whole:L], codes[:, whole:L]
                assert torch.equal(y[:, whole:], a) or torch.equal(y[:, whole:], c), L
    L = lengths[-1]
    before = dm.kv_read_q8(cache, at, L)
    append(5, L)
    after = dm.kv_read_q8(cache, at, L)
    whole = L // BLOCK
    assert all(torch.equal(x, y) for x, y in zip(before, after))
    # from their codes, whatever a read at this length takes from the tail
    far = torch.full((B,), whole * BLOCK + 17, dtype=torch.int32, device=device)
    for x, y in zip(before, dm.kv_read_q8(cache, far, whole * BLOCK)):
        assert torch.equal(x[:, :, :whole * BLOCK], y)
