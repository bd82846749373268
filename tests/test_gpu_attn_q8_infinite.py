"""An infinite value in the tail of an 8-bit cache: the rows that see it, whose weight for
it is positive, are infinite in its feature with its sign, however many parts a head's
blocks are cut into."""
from __future__ import annotations

import pytest
import torch

from tests.kv8_util import D, DTYPES, SLOTS
from tests.test_gpu_attn_q8 import _case

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("bad", [float("inf"), float("-inf")])
@pytest.mark.parametrize("T,Hq,Hkv", [(1, 1, 1), (1, 8, 2), (3, 2, 1), (5, 4, 2), (16, 1, 1), (8, 4, 1), (16, 8, 2)])
@pytest.mark.parametrize("lens", [[30], [130], [200, 300], [650, 700, 1100], [4000]])
def test_sign_of_an_infinite_value(device, dtype, bad, T, Hq, Hkv, lens):
    import dflash_mlx as dm

    cache, lens_d, k, v, q, proj, _ = _case(device, dtype, T, Hq, Hkv, lens, 4032, 3, False, qstd=0.2)
    rep = Hq // Hkv
    for b, L in enumerate(lens):
        cache.tail_vt[b, 0, 9, (L + T // 2) % SLOTS] = bad
    got = dm.attn_verify_q8(q.to(device), cache, lens_d, proj.to(device)).cpu().view(len(lens), T, Hq, D)
    hit = torch.zeros(got.shape, dtype=torch.bool)
    hit[:, T // 2:, :rep, 9] = True
    assert (got[hit] == bad).all()
    assert torch.isfinite(got[~hit].float()).all()
