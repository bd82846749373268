"""Draft blocks that carry a sequence's length past the end of an 8-bit cache: the
positions that it holds read and attend as those of one that ends there, the last block
from its codes, whichever call looks at it first."""
from __future__ import annotations

import pytest
import torch

from tests.kv8_util import BLOCK, D, DTYPES, EPS, THETA, attention_error, expected_read, loaded, proj_rows, random_kv, raw

pytestmark = pytest.mark.gpu

HQ, HKV, SMAX = 4, 2, 192


def _run(device, dtype, starts, T):
    """Sequences loaded up to starts[b], T drafts appended there: (cache, histories)."""
    import dflash_mlx as dm

    B = len(starts)
    k, v = random_kv(B, HKV, SMAX, seed=T, spread=False)
    cache, lens = loaded(device, k, v, starts, SMAX, dtype, fill=0)
    rows = proj_rows(B, T, HQ, HKV, seed=6)
    w = torch.ones(D, dtype=torch.bfloat16, device=device)
    flags = torch.zeros(B, dtype=torch.int32, device=device)
    prep = lambda x, at, prompt=False: dm.attn_prep_q8(  # noqa: E731
        x.to(device), w, w, at, cache, num_heads=HQ, rot_dims=32, rope_base=THETA, eps=EPS, prompt=prompt, overflow=flags)
    prep(rows, lens)
    assert flags.tolist() == [int(L + T > SMAX) for L in starts]
    for b, L in enumerate(starts):  # what the tail has of the new positions
        p = torch.arange(L, min(L + T, SMAX))
        k[b, :, p] = cache.tail_k[b, :, p % 128].cpu()
        v[b, :, p] = cache.tail_vt[b, :, :, p % 128].transpose(1, 2).cpu()
    return cache, k, v, prep


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,starts", [(16, [191, 190, 180, 177, 176]), (5, [188, 187, 191])])
@pytest.mark.parametrize("prompt", [False, True])
def test_lengths_past_the_end(device, dtype, T, starts, prompt):
    import dflash_mlx as dm

    cache, k, v, prep = _run(device, dtype, starts, T)
    lens = [L + T for L in starts]
    at = torch.tensor(lens, dtype=torch.int32, device=device)

    def check_read():
        for x, got in zip((k, v), dm.kv_read_q8(cache, at, SMAX)):
            for b in range(len(lens)):
                assert torch.equal(got[b].cpu(), expected_read(x[b], SMAX, 0, SMAX, dtype)), b

    check_read()  # the last block waits for its codes
    rows = proj_rows(len(starts), 4, HQ, HKV, seed=8)
    q = prep(rows, at, prompt)
    check_read()
    attend = dm.attn_prefill_q8 if prompt else dm.attn_verify_q8
    got = attend(q, cache, at, rows.to(device)).cpu()
    ends = [(SMAX, SMAX // BLOCK)] * len(lens)
    assert attention_error(got, q.cpu(), list(k), list(v), rows, [SMAX] * len(lens), ends, dtype, D ** -0.5) <= 1.0


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("prompt", [False, True])
def test_lengths_that_no_draft_leads_to(device, dtype, prompt):
    """More than 16 past the end: nothing is written."""
    cache, k, v, prep = _run(device, dtype, [170, 100], 16)
    before = raw(cache)
    prep(proj_rows(2, 4, HQ, HKV, seed=8), torch.tensor([SMAX + 17, 2 ** 31 - 1], dtype=torch.int32, device=device), prompt)
    assert all(torch.equal(a, b) for a, b in zip(before, raw(cache)))
