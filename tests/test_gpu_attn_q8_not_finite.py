"""Values that are not finite in the tail of an 8-bit cache, in the verify attention of
up to 16 and of up to 64 query rows a key/value head: in heads that one workgroup has to
itself, in heads cut into parts, and where a workgroup goes through several heads of
which only some hold one.  Rows that see the value are not finite in its feature; every
other output keeps its bits."""
from __future__ import annotations

import pytest
import torch

from tests.kv8_util import D, DTYPES, SLOTS
from tests.test_gpu_attn_q8 import _case

pytestmark = pytest.mark.gpu


def _planted(device, dtype, T, Hq, Hkv, lens, Smax, places, bad):
    """(outputs without, outputs with, hit) [B, T, Hq, D]: `bad` at draft token j, feature d
    of head h's values for every (b, h, j, d)."""
    import dflash_mlx as dm

    cache, lens_d, k, v, q, proj, _ = _case(device, dtype, T, Hq, Hkv, lens, Smax, 3, False)
    q, proj = q.to(device), proj.to(device)
    attend = lambda: dm.attn_verify_q8(q, cache, lens_d, proj).cpu().view(len(lens), T, Hq, D)  # noqa: E731
    clean = attend()
    hit = torch.zeros(clean.shape, dtype=torch.bool)
    rep = Hq // Hkv
    at = [[], [], [], []]
    for b, h, j, d in places:
        for x, y in zip(at, (b, h, d, (lens[b] + j) % SLOTS)):
            x.append(y)
        hit[b, j:, h * rep:(h + 1) * rep, d] = True
    cache.tail_vt[tuple(torch.tensor(x, device=device) for x in at)] = bad
    return clean, attend(), hit


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
@pytest.mark.parametrize("T,Hq,Hkv", [(4, 2, 2), (6, 4, 2), (16, 1, 1), (12, 4, 2), (16, 4, 2), (16, 16, 4)])
@pytest.mark.parametrize("lens", [[40], [120, 130], [1500, 63, 900]])
def test_rows_that_see_the_value(device, dtype, bad, T, Hq, Hkv, lens):
    places = [(b, Hkv - 1, j, d) for b in range(len(lens)) for j, d in ((1, 5), (3, 17), (3, 127))]
    clean, got, hit = _planted(device, dtype, T, Hq, Hkv, lens, 1536, places, bad)
    assert torch.isfinite(clean.float()).all()
    assert not torch.isfinite(got[hit].float()).any()
    assert torch.equal(got[~hit], clean[~hit])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,Hq,Hkv,B", [
    (1, 4, 4, 300),    # eight rows at most of over a thousand heads: two waves a workgroup
    (4, 2, 1, 700),    # eight waves
    (10, 2, 2, 290),
    (16, 4, 2, 330),   # 32 rows
    (16, 8, 2, 300),   # 64 rows
])
def test_heads_that_share_a_workgroup(device, dtype, T, Hq, Hkv, B):
    """More heads than workgroups, every third of them with a NaN."""
    lens = [(29 * i) % 115 for i in range(B)]
    places = [(i // Hkv, i % Hkv, 0, (7 * i) % D) for i in range(B * Hkv) if i % 3 == 1]
    clean, got, hit = _planted(device, dtype, T, Hq, Hkv, lens, 192, places, float("nan"))
    assert torch.isfinite(clean.float()).all()
    assert got[hit].isnan().all()
    assert torch.equal(got[~hit], clean[~hit])
